// Block-sparse attention: every query reads the keys of the `topk` blocks that a cheap score selects for it.
//
//   c_j   = mean of the unmasked keys of block j (block = 32, 64 or 128 consecutive keys)
//   s_ij  = (sum of q_i over the query heads that share the kv head) . c_j
//   B_i   = the topk blocks of largest s_ij among those with an unmasked key, ties to the lower index
//   o_i   = softmax over the unmasked keys of B_i of (scale q_i . k), times v;  0 where there is no such key
//
// The score is linear in q, so the heads of a group are summed first and the selection is one per (query, kv head).
//
// Which block wins must not depend on the order of a sum: scores are 64-bit (a mean of bf16 / fp16 values in 64 bits is exact up to
// its division, and two blocks that are not equal differ by far more than 2^-50 of a score).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "conv_common.h"

namespace yl {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BA_MAX_BLOCKS = 4096;  // key blocks per image: scores of a row in the registers of 8 (many queries) or 16 waves
constexpr int BA_MAX_TOPK = 64;
constexpr int SCORE_MAX_NQ = 4;      // so few queries are scored by the wave that has the mean

// Over the four lanes that share lane & 15 (an MFMA column): v_permlane32_swap / v_permlane16_swap of a register with itself leave
// the two halves' (row pairs') values side by side -- no LDS round trip.
template <typename F>
__device__ __forceinline__ unsigned quad_bits(unsigned x, F f) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  u2 p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = f(p[0], p[1]);
  p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return f(p[0], p[1]);
}
__device__ __forceinline__ float quad_max(float x) {
  return __uint_as_float(quad_bits(__float_as_uint(x), [](unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float quad_min(float x) {
  return __uint_as_float(quad_bits(__float_as_uint(x), [](unsigned a, unsigned b) { return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float quad_sum(float x) {
  return __uint_as_float(quad_bits(__float_as_uint(x), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ int quad_sum(int x) {
  return (int)quad_bits((unsigned)x, [](unsigned a, unsigned b) { return a + b; });
}
__device__ __forceinline__ unsigned quad_or(unsigned x) {
  return quad_bits(x, [](unsigned a, unsigned b) { return a | b; });
}

// Element (b, t, h, c) of a tensor of heads: p + b sb + token(t) st + h sh + (c / 8) sc + c % 8.  Dense tensors: sc = 8, token(t) = t.
// The network's maps (yl_internal.h): a plane per 8 channels, st = 8, sc = a plane, and a guard pixel behind every W tokens.
struct Heads {
  const void* p;
  long long sb, st, sh, sc;
};

struct BlockArgs {
  Heads q, k, v, o;
  int W;  // tokens of a row of the map, 0: no rows
  int batch, nq, nk, heads, kv, group;  // group = heads / kv
  int dk, dv, block, nb, topk;
  const uint8_t* mask;  // [batch][nk], row stride mask_stride; nullptr: every key may be read
  long long mask_stride;
  float scale;
  double* mean;   // [batch][kv][nb][dk]
  double* score;  // few queries: [batch][kv][nq][nb]
  __bf16* split;  // the means as two bf16, in the order the matrix pipe takes them (split_at); nbp = nb rounded up to 16, dkp = dk to 32
  float* norm;    // [batch][kv][nb]: no less than the 2-norm of a mean
  int nbp, dkp;
  float part_err; // what two bf16 for each factor may leave out of a score, relative to the product of the 2-norms
  float head_err; // what the fp32 sum of a group's query heads may be off by, relative to the 2-norm over all of them
  unsigned magic; // 2^32 / group, rounded up: f / group = mulhi(f, magic) for f * group < 2^32
  int* count;     // [batch][nb]: unmasked keys of a block
  int* picked;    // [batch][kv][nq][topk]
};

__device__ __forceinline__ int token(const BlockArgs& a, int t) { return a.W ? t + t / a.W : t; }
// channels 0..7 of (b, t, h); chunk c of eight lies c * x.sc further on
template <typename T>
__device__ __forceinline__ T* head_ptr(const BlockArgs& a, const Heads& x, int b, int t, int h) {
  return static_cast<T*>(const_cast<void*>(x.p)) + b * x.sb + token(a, t) * x.st + h * x.sh;
}

// ------------------------------------------------------------------------------------------------ block means
// value x as two bf16: |x - hi| <= 2^-8 |x|, x = hi + lo up to 2^-17 |x|
__device__ __forceinline__ void split2(float x, __bf16* hi, __bf16* lo) {
  *hi = (__bf16)x;
  *lo = (__bf16)(x - (float)*hi);
}
// At least the 2-norm, from the sum of up to 2^17 squares: those below 2^-126 may have been lost, 2^-54.5 of a norm at most.
__device__ __forceinline__ float norm_of(float squares) { return sqrtf(squares) + 0x1p-54f; }
__device__ __forceinline__ double shfl_xor_d(double x, int o) { return __shfl_xor(x, o); }

// Where the upper half of dim d of block j's mean lies among [batch][kv][nbp / 16][dkp / 32][2][64 lanes][8]: lane (block j % 16, dims
// 8 g .. of 32) of an MFMA operand; the lower half 512 further.  A wave's fragment is then 1 KiB in a row (row by row, 64 bytes of each
// row, the fragment reads took 18 of 34 us of a selection on 80x80 maps).
__device__ __forceinline__ long long split_at(const BlockArgs& a, int bh, int j, int d) {
  return (((long long)bh * (a.nbp >> 4) + (j >> 4)) * (a.dkp >> 5) + (d >> 5)) * 1024 + (((d >> 3) & 3) * 16 + (j & 15)) * 8 + (d & 7);
}

// One wave per (image, kv head, block): lane = (key lane, 8 dims), 64 / CP key lanes (CP: dk / 8 rounded up to a power of two); the
// lanes of a dim chunk exchange halves, then quarters, ... of their sums, so a wave reduces with 7 exchanges instead of 24.
// SCORE: few queries -- the wave that has a block's mean also scores it, and no mean is stored.
// 8 heads x 65536 keys of 64 (67 MB) 18 us, 3700 GB/s: the loads, and beside them 850 vector instructions of a wave (conversions to and
// sums in 64 bits), which take up 45 % of the SIMDs' cycles.
// That wave's part: score[i * step] of the queries, *count keys.
template <typename T, int CP, bool SCORE>
__device__ __forceinline__ void block_mean(const BlockArgs& a, int bh, int j, int lane, double* score, int step, int* count) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  constexpr int KL = 64 / CP;
  const int h = bh % a.kv, b = bh / a.kv;
  const int c = lane % CP, kl = lane / CP;
  const int k0 = j * a.block, kn = min(a.block, a.nk - k0);
  const T* kp = static_cast<const T*>(a.k.p) + b * a.k.sb + h * a.k.sh + c * a.k.sc;
  const uint8_t* mp = a.mask ? a.mask + b * a.mask_stride + k0 : nullptr;
  double acc[8] = {};
  int n = 0;
  for (int i0 = kl; i0 < kn; i0 += 8 * KL) {  // eight keys of a lane in flight
    t8 x[8];
    bool ok[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * KL;
      ok[u] = i < kn && (!mp || mp[i]);
      x[u] = t8{};
      if (ok[u] && c * 8 < a.dk) x[u] = *reinterpret_cast<const t8*>(kp + token(a, k0 + i) * a.k.st);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      n += ok[u];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += (double)(float)x[u][e];
    }
  }
#pragma unroll
  for (int o = CP; o < 64; o <<= 1) n += __shfl_xor(n, o);
  // lane bits CP, 2 CP, 4 CP: the partner's half of the dims comes here, the other half goes there
  int d0 = 0;
#pragma unroll
  for (int step = 0; step < 3; ++step) {
    const int o = CP << step, half = 4 >> step;
    if (o < 64) {
      const bool up = lane & o;
#pragma unroll
      for (int e = 0; e < half; ++e) {
        const double give = up ? acc[e] : acc[half + e], keep = up ? acc[half + e] : acc[e];
        acc[e] = keep + shfl_xor_d(give, o);
      }
      d0 += up ? half : 0;
    }
  }
#pragma unroll
  for (int o = CP * 8; o < 64; o <<= 1) acc[0] += shfl_xor_d(acc[0], o);  // (all eight dims are one per lane by now)
  constexpr int LEFT = CP == 16 ? 2 : 1;  // dims a lane ends up with
  const bool mine = kl < 8 && c * 8 < a.dk;
  double mean[LEFT];
#pragma unroll
  for (int e = 0; e < LEFT; ++e) mean[e] = n ? acc[e] / n : 0.0;
  if constexpr (SCORE) {
    for (int i = 0; i < a.nq; ++i) {
      double s = 0;
      if (mine)
#pragma unroll
        for (int e = 0; e < LEFT; ++e) {
          double q = 0;
          for (int g = 0; g < a.group; ++g)
            q += (double)(float)head_ptr<const T>(a, a.q, b, i, h * a.group + g)[c * a.q.sc + d0 + e];
          s += q * mean[e];
        }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) s += shfl_xor_d(s, o);
      if (lane == 0) score[(long long)i * step] = n ? s : __builtin_nan("");
    }
    if (lane == 0 && count) *count = n;
  } else {
    float norm = 0.f;
    if (mine)
#pragma unroll
      for (int e = 0; e < LEFT; ++e) {
        const int d = c * 8 + d0 + e;
        a.mean[((long long)bh * a.nb + j) * a.dk + d] = mean[e];
        const float f = (float)mean[e];
        __bf16 hi, lo;
        split2(f, &hi, &lo);
        __bf16* at = a.split + split_at(a, bh, j, d);
        at[0] = hi;
        at[512] = lo;
        norm += f * f;
      }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) norm += __shfl_xor(norm, o);
    if (lane < a.dkp - a.dk) {  // the dims behind the last: zeros
      __bf16* at = a.split + split_at(a, bh, j, a.dk + lane);
      at[0] = at[512] = (__bf16)0.f;
    }
    if (lane == 0) {
      a.norm[(long long)bh * a.nb + j] = norm_of(norm);
      if (count) *count = n;
    }
  }
}
template <typename T, int CP, bool SCORE>
__global__ __launch_bounds__(256) void block_mean_kernel(BlockArgs a) {
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6);  // (below 2^31, as the blocks are: no 64-bit division)
  if (unit >= (unsigned)(a.batch * a.kv * a.nb)) return;
  const int bh = (int)(unit / (unsigned)a.nb), j = (int)(unit - (unsigned)bh * (unsigned)a.nb);
  block_mean<T, CP, SCORE>(a, bh, j, threadIdx.x & 63, SCORE ? a.score + (long long)bh * a.nq * a.nb + j : nullptr, a.nb,
                           bh % a.kv == 0 ? a.count + (bh / a.kv) * a.nb + j : nullptr);
}

// ------------------------------------------------------------------------------------------------ selection
// Scores in the order of unsigned integers; 0: the block cannot be selected.  NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ unsigned long long order_key(double s, bool can) {
  if (!can) return 0;
  if (s != s) s = -__builtin_inf();
  const unsigned long long b = (unsigned long long)__double_as_longlong(s + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// sum over the 64 lanes, the same in all of them (row shifts, row broadcasts: no LDS round trips)
__device__ __forceinline__ int wave_sum(int c) {
  c += __builtin_amdgcn_update_dpp(0, c, 0x111, 0xF, 0xF, false);
  c += __builtin_amdgcn_update_dpp(0, c, 0x112, 0xF, 0xF, false);
  c += __builtin_amdgcn_update_dpp(0, c, 0x114, 0xF, 0xF, false);
  c += __builtin_amdgcn_update_dpp(0, c, 0x118, 0xF, 0xF, false);
  c += __builtin_amdgcn_update_dpp(0, c, 0x142, 0xA, 0xF, false);
  c += __builtin_amdgcn_update_dpp(0, c, 0x143, 0xC, 0xF, false);
  return __builtin_amdgcn_readlane(c, 63);
}

__device__ __forceinline__ unsigned wave_or(unsigned c) {
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x111, 0xF, 0xF, false);
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x112, 0xF, 0xF, false);
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x114, 0xF, 0xF, false);
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x118, 0xF, 0xF, false);
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x142, 0xA, 0xF, false);
  c |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)c, 0x143, 0xC, 0xF, false);
  return (unsigned)__builtin_amdgcn_readlane((int)c, 63);
}

// the larger of each pair of 16-bit numbers over the 64 lanes
__device__ __forceinline__ unsigned wave_max2(unsigned c) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  auto max2 = [](unsigned x, int y) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
  };
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x111, 0xF, 0xF, false));
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x112, 0xF, 0xF, false));
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x114, 0xF, 0xF, false));
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x118, 0xF, 0xF, false));
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x142, 0xA, 0xF, false));
  c = max2(c, __builtin_amdgcn_update_dpp(0, (int)c, 0x143, 0xC, 0xF, false));
  return (unsigned)__builtin_amdgcn_readlane((int)c, 63);
}

// The same over a workgroup's NW waves (all of them call), through two small buffers of LDS in turn: one barrier each.
template <int NW>
struct Waves {
  int (*red)[NW];  // [2][NW]
  int lane, wave, turn;
  __device__ __forceinline__ void put(int x) {
    turn ^= 1;
    if (lane == 0) red[turn][wave] = x;
    __syncthreads();
  }
  __device__ __forceinline__ int sum(int x) {
    x = wave_sum(x);
    if constexpr (NW == 1) return x;
    put(x);
    return wave_sum(lane < NW ? red[turn][lane] : 0);
  }
  __device__ __forceinline__ unsigned any(unsigned x) {
    x = wave_or(x);
    if constexpr (NW == 1) return x;
    put((int)x);
    return wave_or(lane < NW ? (unsigned)red[turn][lane] : 0u);
  }
  __device__ __forceinline__ int before(int x) {  // sum over the waves ahead of this one
    if constexpr (NW == 1) return 0;
    put(wave_sum(x));
    return wave_sum(lane < wave ? red[turn][lane] : 0);
  }
};

// The n-th largest of the keys that the lanes hold (0: none), by its bits, upper word first: the lower words are looked at where the
// upper ones leave it open (ties).
template <int NW, int NI>
__device__ __forceinline__ unsigned long long nth_key(const unsigned long long (&key)[NI], int n, Waves<NW>& ws) {
  unsigned any = 0, none = 0;  // bits set in some key, clear in some key
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    any |= (unsigned)(key[i] >> 32);
    none |= ~(unsigned)(key[i] >> 32);
  }
  any = ws.any(any);
  const unsigned differ = any & ws.any(none);  // bits that all keys share need no decision
  unsigned vh = any & ~differ, vl = 0;
  bool exact = false;
  for (unsigned left = differ; left && !exact;) {
    const unsigned bit = 1u << (31 - __clz(left));
    left &= ~bit;
    int c = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) c += (unsigned)(key[i] >> 32) >= (vh | bit);
    c = ws.sum(c);
    if (c >= n) vh |= bit;
    exact = c == n;
  }
  for (int bit = 31; bit >= 0 && !exact; --bit) {
    const unsigned long long t = (unsigned long long)vh << 32 | vl | 1u << bit;
    int c = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) c += key[i] >= t;
    c = ws.sum(c);
    if (c >= n) vl |= 1u << bit;
    exact = c == n;
  }
  return (unsigned long long)vh << 32 | vl;
}

// NW waves: lane holds the keys of blocks 64 (NI wave + i) + lane (0 behind the last) -> the topk largest in ascending order; of equal
// ones the first.
template <int NW, int NI>
__device__ __forceinline__ void pick_row(const unsigned long long (&key)[NI], int topk, Waves<NW>& ws, int* out) {
  const int lane = ws.lane;
  int can = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) can += key[i] != 0;
  const int n = min(topk, ws.sum(can));
  if (n > 0) {
    const unsigned long long v = nth_key(key, n, ws);
    int over = 0, same = 0;  // keys > v, keys equal to v
#pragma unroll
    for (int i = 0; i < NI; ++i) over += key[i] > v, same += key[i] == v;
    int ties = n - ws.sum(over), at = 0;  // of the equal keys the first `ties` belong to the set
    if constexpr (NW > 1) {
      ties = max(0, ties - ws.before(same));
      const int mine = wave_sum(over) + min(ties, wave_sum(same));
      at = ws.before(lane == 0 ? mine : 0);
    }
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const unsigned long long eq = __ballot(key[i] == v);
      const bool take = key[i] > v || (key[i] == v && __popcll(eq & below) < ties);
      ties -= min(ties, (int)__popcll(eq));
      const unsigned long long got = __ballot(take);
      if (take) out[at + __popcll(got & below)] = (ws.wave * NI + i) * 64 + lane;
      at += __popcll(got);
    }
  }
  for (int t = n + ws.wave * 64 + lane; t < topk; t += 64 * NW) out[t] = -1;
}

// One wave: the exact scores of one (image, kv head, query) from the 64-bit means, as keys of blocks j0 + 64 x + lane.  qs: dk doubles
// of LDS.
template <typename T, int NI>
__device__ __forceinline__ void exact_keys(const BlockArgs& a, int bh, int i, int j0, int lane, double* qs, unsigned long long (&key)[NI]) {
  const int h = bh % a.kv, b = bh / a.kv;
  for (int d = lane; d < a.dk; d += 64) {
    double s = 0;
    for (int g = 0; g < a.group; ++g)
      s += (double)(float)head_ptr<const T>(a, a.q, b, i, h * a.group + g)[(d >> 3) * a.q.sc + (d & 7)];
    qs[d] = s;
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int x = 0; x < NI; ++x) {
    const int j = j0 + x * 64 + lane;
    key[x] = 0;
    if (j < a.nb) {
      double s = 0;
      const double* m = a.mean + ((long long)bh * a.nb + j) * a.dk;
#pragma unroll 2
      for (int d = 0; d < a.dk; ++d) s += qs[d] * m[d];
      key[x] = order_key(s, a.count[b * a.nb + j] > 0);
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// Few queries: the scores are there.  NW waves per (image, kv head, query), up to 256 NW blocks.  Nothing here but latency: 256 blocks 5,
// 1024 blocks 8.4 us (by one wave, 16 to a lane, 11.6).
template <int NW>
__global__ __launch_bounds__(64 * NW) void block_select_kernel(BlockArgs a) {
  constexpr int NI = 4;
  __shared__ int red[2][NW];
  Waves<NW> ws{red, (int)threadIdx.x & 63, (int)threadIdx.x >> 6, 0};
  const long long row = blockIdx.x;  // (b * kv + h) * nq + i
  const int b = (int)(blockIdx.x / (unsigned)a.nq / (unsigned)a.kv);
  unsigned long long key[NI];
  double s[NI];
  int n[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) {  // (all in flight together)
    const int at = (ws.wave * NI + x) * 64 + ws.lane, j = min(at, a.nb - 1);
    s[x] = a.nb ? a.score[row * a.nb + j] : 0.0;
    n[x] = at < a.nb ? a.count[b * a.nb + j] : 0;
  }
#pragma unroll
  for (int x = 0; x < NI; ++x) key[x] = order_key(s[x], n[x] > 0);
  pick_row(key, a.topk, ws, a.picked + row * a.topk);
}

// Few queries and up to 16 short blocks, one to a wave: one workgroup per (image, kv head) does both, in one launch.  Call, one launch / two:
// one query, 8 kv heads, 7 blocks of 64 x 64 10.2 / 12.7 us, 16 blocks 10.2 / 13.1; two blocks to a wave 18.8 / 13.0, and 30.9 / 13.3 of 128 x 128.
constexpr int SMALL_BLOCKS = 16, SMALL_BLOCK = 64 * 128;
template <typename T, int CP>
__global__ __launch_bounds__(1024) void block_select_small_kernel(BlockArgs a) {
  __shared__ double score[SCORE_MAX_NQ][SMALL_BLOCKS];
  __shared__ int count[SMALL_BLOCKS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bh = (int)blockIdx.x;
  if (wave < a.nb) block_mean<T, CP, true>(a, bh, wave, lane, &score[0][wave], SMALL_BLOCKS, &count[wave]);
  __syncthreads();
  if (wave >= a.nq) return;
  Waves<1> ws{nullptr, lane, 0, 0};
  const unsigned long long key[1] = {lane < a.nb ? order_key(score[wave][lane], count[lane] > 0) : 0};
  pick_row(key, a.topk, ws, a.picked + ((long long)bh * a.nq + wave) * a.topk);
}

// Scores of 16 queries with the means of blocks 16 t0 .. 16 (t0 + NT) on the matrix pipe: lane (query n, group g) gets those of
// blocks 16 (t0 + t) + 4 g + r, and its share of the squared norms of the query (qq) and of all its heads (hh).  qp: the query's first
// head; bh: its means.
template <typename T, int NT>
__device__ __forceinline__ void score_tiles(const BlockArgs& a, int bh, const T* qp, int t0, int lane, f32x4 (&s)[NT], float& qq, float& hh) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  qq = 0.f, hh = 0.f;
  const __bf16* sp = a.split + split_at(a, bh, 0, 0) + lane * 8;
  for (int c0 = 0; c0 < a.dkp; c0 += 32) {
    const int c = c0 + g * 8;
    float q[8] = {};
    if (c < a.dk) {
      if (a.group == 1) {  // (the loop below would ask for it four times: 80x80 maps 31.9 us instead of 30.6)
        const t8 x = *reinterpret_cast<const t8*>(qp + (c >> 3) * a.q.sc);
#pragma unroll
        for (int d = 0; d < 8; ++d) q[d] = (float)x[d];
      } else {
        for (int e0 = 0; e0 < a.group; e0 += 4) {  // four heads' loads in flight together
          t8 x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const t8*>(qp + min(e0 + e, a.group - 1) * a.q.sh + (c >> 3) * a.q.sc);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e0 + e < a.group)
#pragma unroll
              for (int d = 0; d < 8; ++d) q[d] += (float)x[e][d], hh = __builtin_fmaf((float)x[e][d], (float)x[e][d], hh);
        }
      }
    }
    bf16x8 qh, ql;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      __bf16 hi, lo;
      split2(q[d], &hi, &lo);
      qh[d] = hi, ql[d] = lo;
      qq += q[d] * q[d];
    }
    constexpr int TB = NT < 8 ? NT : 8;  // tiles whose loads are in flight together
#pragma unroll
    for (int u0 = 0; u0 < NT; u0 += TB) {
      if ((t0 + u0) * 16 >= a.nb) break;
      bf16x8 mh[TB], ml[TB];
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        const unsigned m = ((unsigned)min(t0 + u0 + t, (a.nbp >> 4) - 1) * (unsigned)(a.dkp >> 5) + (unsigned)(c0 >> 5)) * 1024u;
        mh[t] = *reinterpret_cast<const bf16x8*>(sp + m);
        ml[t] = *reinterpret_cast<const bf16x8*>(sp + m + 512);
      }
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        s[u0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mh[t], qh, s[u0 + t], 0, 0, 0);
        s[u0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ml[t], qh, s[u0 + t], 0, 0, 0);
        s[u0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mh[t], ql, s[u0 + t], 0, 0, 0);
        s[u0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ml[t], ql, s[u0 + t], 0, 0, 0);
      }
    }
  }
}
// what such a score may be off by; qn, hn, cn: the norms of the query, of all its heads and of the largest mean
__device__ __forceinline__ float score_error(const BlockArgs& a, float qn, float hn, float cn) {
  return ((a.part_err + 4.f * a.dk / 16777216.f) * qn + a.head_err * hn) * cn + (qn + cn) * 2e-36f + 1e-30f;
}

// One wave: of nmay <= 16 candidates (lane c < nmay: block mj) the `need` with the largest 64-bit scores, as a mask of lanes; of equal
// scores the lower block first.  qsum: dk doubles of LDS.
template <typename T>
__device__ __forceinline__ unsigned long long choose_exact(const BlockArgs& a, int bh, int i, int lane, int nmay, int need, int mj, double* qsum) {
  const int h = bh % a.kv, b = bh / a.kv;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int d = lane + 64 * x;
    if (d < a.dk) {
      double q = 0;
      for (int e = 0; e < a.group; ++e) q += (double)(float)head_ptr<const T>(a, a.q, b, i, h * a.group + e)[(d >> 3) * a.q.sc + (d & 7)];
      qsum[d] = q;
    }
  }
  __builtin_amdgcn_wave_barrier();
  double mine = 0;
  for (int c0 = 0; c0 < nmay; c0 += 4) {  // four candidates at a time, sixteen lanes each
    const int j = __shfl(mj, min(c0 + (lane >> 4), nmay - 1));
    const double* m = a.mean + ((long long)bh * a.nb + j) * a.dk;
    double x = 0;
    for (int d = lane & 15; d < a.dk; d += 16) x += qsum[d] * m[d];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) x += shfl_xor_d(x, o);
    const double y = __shfl(x, (lane - c0 & 3) * 16);
    if (lane >= c0 && lane < c0 + 4) mine = y;
  }
  __builtin_amdgcn_wave_barrier();
  int before = 0;  // candidates in front of this lane's
  for (int x = 0; x < nmay; ++x) {
    const double v = __shfl(mine, x);
    before += v > mine || (v == mine && x < lane);
  }
  return __ballot(lane < nmay && before < need);
}

// Many queries, up to 16 NT blocks: a wave scores 16 queries at once on the matrix pipe, in less than 64 bits, and decides only what
// that can decide.  q (summed over the group) and the means are split into two bf16 each; all four products together are off by less than
//   score_error = (part_err + 4 dk 2^-24) |q| |c|     (|.| the 2-norms; 4 dk 2^-24: an fp32 sum of 4 dk terms, the fourth below 2^-16)
// of a score, part_err = 2^-17 for what the mean's two parts leave out, 2^-17 for what q's leave (none of one head's 8 or 11 bits) and a
// twentieth of that for the mean's own rounding to fp32 (2^-24) and products of these (and, where a part is not a normal number any more,
// dk 2^-126 times the other norm; near the ends of fp32's range nothing is decided here).  Without the product of the two lower parts
// part_err is 2^-16 more, and 2 x 16384 queries x 256 blocks, four heads to one, took 40 instead of 39 us.  The sum of a group's n heads
// is off by up to (n - 1) 2^-24 sum |q_h| in each dim, hence a score by up to (n - 1) sqrt(n) 2^-24 |q_1 .. q_n| |c| more: heads may
// cancel, so this goes by the norm over all of them.  Lane (query n, group g) holds the scores of blocks 16 t + 4 g + r; the cut that
// leaves topk of them over it is found by bisection, 16 queries in step.  Where the last block over the cut
// and the first under it are more than 2 err apart -- all but a few in a thousand -- the order is the exact one's; the other queries
// (ties, NaN and infinities among them) are scored in 64 bits.
// 12 heads x 6400 queries x 100 blocks 27 us, 48 x 1600 x 25 17 us, 2 x 16384 x 256 (four query heads to one) 38 us: 1800, 1100 and 4000
// vector instructions of a wave, about half of them the bisection's comparisons, issued in 42, 37 and 31 % of the cycles -- the steps of
// the bisection wait for one another, and there are few waves beside each other to fill in.
template <typename T, int NT>
__global__ __launch_bounds__(256, NT <= 8 ? 4 : 2) void block_score_kernel(BlockArgs a, int qtiles) {
  __shared__ double qs[4][128];
  constexpr int NWORD = (NT + 1) / 2;  // 32 blocks to a word
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  const unsigned unit = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x) * 4u + (unsigned)wave;  // (below 2^31: the rows are)
  if (unit >= (unsigned)(a.batch * a.kv) * (unsigned)qtiles) return;  // (no barrier below: waves are on their own)
  const int bh = (int)(unit / (unsigned)qtiles), qt = (int)(unit - (unsigned)bh * (unsigned)qtiles), h = bh % a.kv, b = bh / a.kv;
  const int i = qt * 16 + n;
  const bool live = i < a.nq;
  const float ninf = -__builtin_huge_valf();

  // how many keys each block has to read, |c| -- asked for ahead of everything else
  int cnt[(NWORD + 1) / 2];
  float norm[(NWORD + 1) / 2];
#pragma unroll
  for (int w = 0; w < (NWORD + 1) / 2; ++w) {
    const int j = min(w * 64 + lane, a.nb - 1);
    cnt[w] = a.count[b * a.nb + j];
    norm[w] = a.norm[(long long)bh * a.nb + j];
    if (w * 64 + lane >= a.nb) cnt[w] = 0, norm[w] = 0.f;
  }
  // ---- scores
  f32x4 s[NT];
  float qq, hh;
  score_tiles<T, NT>(a, bh, head_ptr<const T>(a, a.q, b, live ? i : 0, h * a.group), 0, lane, s, qq, hh);
  // ---- which blocks can be selected, how many there are, the largest |c|
  unsigned okw[NWORD];
  int can = 0;
  float big = 0.f;
#pragma unroll
  for (int w = 0; w < NWORD; w += 2) {
    const unsigned long long ok = __ballot(cnt[w / 2] > 0);
    okw[w] = (unsigned)ok;
    if (w + 1 < NWORD) okw[w + 1] = (unsigned)(ok >> 32);
    can += __popcll(ok);
    big = fmaxf(big, norm[w / 2] < __builtin_huge_valf() ? norm[w / 2] : __builtin_huge_valf());  // (NaN: no bound)
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) big = fmaxf(big, __shfl_xor(big, o));
  big = quad_max(big);
  const int take = min(a.topk, can);
  const float qn = norm_of(quad_sum(qq));
  const float err = score_error(a, qn, a.group > 1 ? norm_of(quad_sum(hh)) : 0.f, big);

  // ---- the cut.  Blocks that cannot be selected (and places behind the last) go under every cut
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if ((okw[t >> 1] >> ((t & 1) * 16) & 0xFFFFu) == 0xFFFFu) continue;  // (the same in every lane)
    const unsigned m = okw[t >> 1] >> ((t & 1) * 16 + 4 * g);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[t][r] = m >> r & 1 ? s[t][r] : ninf;
  }
  float hi = ninf;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) hi = __builtin_amdgcn_fmed3f(hi, s[t][r], __builtin_huge_valf());
  hi = quad_max(hi);
  float lo = -1.01f * qn * big - 1e-30f;  // under every score
  // more than `take` scores over lo, fewer over hi.  (Half way: about 12 steps until all 16 queries are done; a straight line between
  // the two counts took 14-16, the counts fall too steeply towards the cut.)
  float cut = ninf;
  bool found = take == can;  // (everything that can be selected is: the cut stays at -inf)
  for (int it = 0; it < 32 && __ballot(!found && live); ++it) {
    const float mid = 0.5f * (lo + hi);
    int c = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) c += s[t][r] > mid;
    c = quad_sum(c);
    if (c == take) cut = found ? cut : mid, found = true;
    lo = c > take && !found ? mid : lo;
    hi = c < take && !found ? mid : hi;
  }
  // Sure where no score lies within err of the cut: the two sides are more than 2 err apart.  (Not so where anything is NaN.)  Only
  // where that fails for some query are the two sides themselves looked for.
  float near = __builtin_huge_valf();
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) near = fminf(near, fabsf(s[t][r] - cut));
  near = quad_min(near);
  const bool fine = qn * big < 1e37f;
  bool sure = take == can || (found && fine && near > err);
  float in = __builtin_huge_valf(), out = ninf;
  if (__ballot(!sure && live)) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool over = s[t][r] > cut;
        in = over ? fminf(in, s[t][r]) : in;
        out = over ? out : fmaxf(out, s[t][r]);
      }
    in = quad_min(in);
    out = quad_max(out);
    sure = sure || (found && fine && in - out > 2.f * err);
  }
  const float up = (found ? out : hi) + 2.f * err, dn = (found ? in : lo) - 2.f * err;   // the band around a cut that is not sure
  const float floor_ = sure ? cut : up;

  // ---- picked blocks as words of 32, the same in every lane of a query; lane g writes the ranks g, g + 4, ... (a lane that wrote its own
  // blocks had up to eight of a word where neighbours are picked together: 9 us of 33)
  int* const row = a.picked + ((long long)bh * a.nq + i) * a.topk;
  unsigned inw[NWORD];
  int at = 0;
#pragma unroll
  for (int w = 0; w < NWORD; ++w) {
    unsigned bits = 0;
#pragma unroll
    for (int t = 2 * w; t < 2 * w + 2 && t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) bits |= (unsigned)(s[t][r] > floor_) << ((t & 1) * 16 + r);
    bits = quad_or(bits << (4 * g));
    inw[w] = take == can ? okw[w] : bits;
    at += __popc(inw[w]);
  }
  if (sure && live)
    for (int t = g; t < a.topk; t += 4) {
      int k = t, j = -1;
      unsigned bits = 0;
#pragma unroll
      for (int w = 0; w < NWORD; ++w) {  // the word that holds rank t
        const int n = __popc(inw[w]);
        if (j < 0) {
          if (k < n) j = w * 32, bits = inw[w];
          else k -= n;
        }
      }
      if (j >= 0)
#pragma unroll
        for (int o = 16; o; o >>= 1) {  // its k-th set bit
          const int n = __popc(bits & ((1u << o) - 1));
          if (k >= n) k -= n, j += o, bits >>= o;
        }
      row[t] = j;
    }
  // the other queries, one after another: 64-bit scores of the blocks next to the cut, or of all where that says too little
  unsigned long long todo = __ballot(!sure && live) & 0xFFFF;
  if (!todo) return;
  unsigned mayw[NWORD];
  int may = 0;
#pragma unroll
  for (int w = 0; w < NWORD; ++w) {
    unsigned bits = 0;
#pragma unroll
    for (int t = 2 * w; t < 2 * w + 2 && t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) bits |= (unsigned)(s[t][r] <= up && s[t][r] >= dn) << ((t & 1) * 16 + r);
    mayw[w] = quad_or(bits << (4 * g)) & okw[w];
    may += __popc(mayw[w]);
  }
  const bool few = fine && may <= 16 && at <= take && at + may >= take;
  while (todo) {
    const int k = __ffsll(todo) - 1;
    todo &= todo - 1;
    const int qi = qt * 16 + k;
    if (!__builtin_amdgcn_readlane((int)few, k)) {
      unsigned long long key[(NT + 3) / 4];
      exact_keys<T>(a, bh, qi, 0, lane, qs[wave], key);
      Waves<1> ws{nullptr, lane, 0, 0};
      pick_row(key, a.topk, ws, a.picked + ((long long)bh * a.nq + qi) * a.topk);
      continue;
    }
    const int nmay = __builtin_amdgcn_readlane(may, k), need = __builtin_amdgcn_readlane(take - at, k);
    int mj = 0, c = 0;  // lane c: candidate c
#pragma unroll
    for (int w = 0; w < NWORD; ++w) {
      unsigned bits = (unsigned)__builtin_amdgcn_readlane((int)mayw[w], k);
      while (bits) {  // (the same in every lane)
        mj = lane == c ? w * 32 + __ffs(bits) - 1 : mj;
        bits &= bits - 1;
        ++c;
      }
    }
    const unsigned long long chosen = choose_exact<T>(a, bh, qi, lane, nmay, need, mj, qs[wave]);
    int* const to = a.picked + ((long long)bh * a.nq + qi) * a.topk;
    int base = 0;
#pragma unroll
    for (int w = 0; w < NWORD; ++w) {
      unsigned bits = (unsigned)__builtin_amdgcn_readlane((int)inw[w], k);
      for (unsigned long long left = chosen; left; left &= left - 1) {
        const int j = __builtin_amdgcn_readlane(mj, __ffsll(left) - 1);
        if (j >> 5 == w) bits |= 1u << (j & 31);
      }
      if (lane < 32 && (bits >> lane & 1)) to[base + __popc(bits & ((1u << lane) - 1))] = w * 32 + lane;
      base += __popc(bits);
    }
    for (int t = base + lane; t < a.topk; t += 64) to[t] = -1;
  }
}

// The same by NW waves (4 or 8) for 16 queries: wave w has blocks 16 NT w .., each step of the bisection adds up their counts through
// LDS.  Then a wave finishes 16 / NW queries, from words of 64 blocks.  What it is for: more blocks than a wave's registers hold scores
// of (16384 queries, 513 blocks, four heads of 64 to one kv head: a wave per query with every score in 64 bits 707 us, this 81; 8192 queries,
// 1024 blocks, eight heads of 128 to one: 1159 and 75 us), and few queries.  Most of it are comparisons: 12 steps over the scores in
// registers.
template <typename T, int NW, int NT>
__global__ __launch_bounds__(64 * NW) void block_score_wide_kernel(BlockArgs a, int qtiles) {
  constexpr int WORDS = NT / 4;  // of a wave
  __shared__ double qs[NW][128];
  __shared__ unsigned long long inw[16][64], mayw[16][64];
  __shared__ int red[2][NW][16], red1[2][NW];
  __shared__ int cand[NW][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  const unsigned unit = (unsigned)xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int bh = (int)(unit / (unsigned)qtiles), qt = (int)(unit - (unsigned)bh * (unsigned)qtiles), h = bh % a.kv, b = bh / a.kv;
  const int i = qt * 16 + n, t0 = wave * NT;
  const bool live = i < a.nq;
  const float ninf = -__builtin_huge_valf(), inf = __builtin_huge_valf();

  // a value per wave and query -> over the waves.  (Two buffers: one barrier is enough)
  int turn = 0;
  auto gather = [&](int x, int* lo, int* hi) __attribute__((always_inline)) {
    turn ^= 1;
    if (g == 0) red[turn][wave][n] = x;
    __syncthreads();
    *lo = red[turn][g][n], *hi = NW == 8 ? red[turn][NW - 4 + g][n] : 0;
  };
  auto sum_all = [&](int x) __attribute__((always_inline)) {
    int p, q;
    gather(x, &p, &q);
    return quad_sum(p + q);
  };
  auto max_all = [&](float x) __attribute__((always_inline)) {
    int p, q;
    gather((int)__float_as_uint(x), &p, &q);
    return quad_max(NW == 8 ? fmaxf(__uint_as_float((unsigned)p), __uint_as_float((unsigned)q)) : __uint_as_float((unsigned)p));
  };

  // ---- which of this wave's blocks can be selected, how many there are in all, the largest |c|; scores
  unsigned long long okw[WORDS];
  int can = 0;
  float big = 0.f;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int j = t0 * 16 + w * 64 + lane;
    const float norm = j < a.nb ? a.norm[(long long)bh * a.nb + j] : 0.f;
    okw[w] = __ballot(j < a.nb && a.count[b * a.nb + min(j, a.nb - 1)] > 0);
    can += __popcll(okw[w]);
    big = fmaxf(big, norm < inf ? norm : inf);  // (NaN: no bound)
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) big = fmaxf(big, __shfl_xor(big, o));
  big = max_all(quad_max(big));
  can = sum_all(can);
  f32x4 s[NT];
  float qq, hh;
  score_tiles<T, NT>(a, bh, head_ptr<const T>(a, a.q, b, live ? i : 0, h * a.group), t0, lane, s, qq, hh);
  const int take = min(a.topk, can);
  const float qn = norm_of(quad_sum(qq));
  const float err = score_error(a, qn, a.group > 1 ? norm_of(quad_sum(hh)) : 0.f, big);

  // ---- the cut, as above
  float hi = ninf;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const unsigned m = (unsigned)(okw[t >> 2] >> ((t & 3) * 16 + 4 * g));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[t][r] = m >> r & 1 ? s[t][r] : ninf;
      hi = fmaxf(hi, s[t][r]);
    }
  }
  hi = max_all(quad_max(hi));
  float lo = -1.01f * qn * big - 1e-30f;
  float cut = ninf;
  bool found = take == can;
  for (int it = 0; it < 32 && __ballot(!found && live); ++it) {  // (the same in every wave)
    const float mid = 0.5f * (lo + hi);
    int c = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) c += s[t][r] > mid;
    c = sum_all(quad_sum(c));
    if (c == take) cut = found ? cut : mid, found = true;
    lo = c > take && !found ? mid : lo;
    hi = c < take && !found ? mid : hi;
  }
  float in = inf, out = ninf;  // the two sides of the cut
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool over = s[t][r] > cut;
      in = over ? fminf(in, s[t][r]) : in;
      out = over ? out : fmaxf(out, s[t][r]);
    }
  in = -max_all(-quad_min(in));
  out = max_all(quad_max(out));
  const bool fine = qn * big < 1e37f, sure = take == can || (found && fine && in - out > 2.f * err);
  const float up = (found ? out : hi) + 2.f * err, dn = (found ? in : lo) - 2.f * err;
  const float floor_ = sure ? cut : up;

  // ---- words of 64 blocks: picked, and in the band around a cut that is not sure
  int at = 0, may = 0;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    unsigned long long over = 0, band = 0;
#pragma unroll
    for (int t = 4 * w; t < 4 * w + 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        over |= (unsigned long long)(s[t][r] > floor_) << ((t & 3) * 16 + r);
        band |= (unsigned long long)(!sure && s[t][r] <= up && s[t][r] >= dn) << ((t & 3) * 16 + r);
      }
    over <<= 4 * g, band <<= 4 * g;
    over = (unsigned long long)quad_or((unsigned)(over >> 32)) << 32 | quad_or((unsigned)over);
    band = (unsigned long long)quad_or((unsigned)(band >> 32)) << 32 | quad_or((unsigned)band);
    over = take == can ? okw[w] : over;
    band &= okw[w];
    at += __popcll(over), may += __popcll(band);
    if (g == 0) inw[n][wave * WORDS + w] = over, mayw[n][wave * WORDS + w] = band;
  }
  at = sum_all(at);
  may = sum_all(may);  // (and the words of all waves are there)
  const bool few = fine && may <= 16 && at <= take && at + may >= take;

  // ---- queries about which that says too little: 64-bit scores of all blocks, by all waves
  const unsigned long long all = __ballot(!sure && !few && live) & 0xFFFF;  // (the same in every wave)
  Waves<NW> ws{red1, lane, wave, 0};
  for (unsigned long long todo = all; todo; todo &= todo - 1) {
    const int k = __ffsll(todo) - 1;
    unsigned long long key[WORDS];
    exact_keys<T>(a, bh, qt * 16 + k, t0 * 16, lane, qs[wave], key);
    const int want = __builtin_amdgcn_readlane(take, k);  // (fewer than can be selected: the others are sure)
    const unsigned long long v = nth_key(key, want, ws);
    int over = 0, same = 0;
#pragma unroll
    for (int x = 0; x < WORDS; ++x) over += key[x] > v, same += key[x] == v;
    int ties = want - ws.sum(over);
    ties = max(0, ties - ws.before(same));
#pragma unroll
    for (int x = 0; x < WORDS; ++x) {
      const unsigned long long eq = __ballot(key[x] == v);
      const bool got = key[x] > v || (key[x] == v && __popcll(eq & ((1ull << lane) - 1)) < ties);
      ties -= min(ties, (int)__popcll(eq));
      const unsigned long long bits = __ballot(got);
      if (lane == 0) inw[k][wave * WORDS + x] = bits;
    }
  }
  if (all) __syncthreads();

  // ---- this wave's two queries: lane l has blocks 64 l ..
  for (int k = 16 / NW * wave; k < 16 / NW * (wave + 1); ++k) {
    const int qi = qt * 16 + k;
    if (qi >= a.nq) break;
    const bool some = __builtin_amdgcn_readlane((int)(!sure && few), k);  // some of the blocks of the band
    auto places = [&](unsigned long long bits, int* total) {  // bits in the lanes before this one
      const int c = __popcll(bits);
      int x = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      *total = __shfl(x, 63);
      return x - c;
    };
    unsigned long long bits = lane < NW * WORDS ? inw[k][lane] : 0;
    if (some) {
      int nmay;
      unsigned long long band = lane < NW * WORDS ? mayw[k][lane] : 0;
      for (int c = places(band, &nmay); band; band &= band - 1) cand[wave][c++] = lane * 64 + __ffsll(band) - 1;
      __builtin_amdgcn_wave_barrier();
      const int mj = cand[wave][max(0, min(lane, nmay - 1))];
      const int need = __builtin_amdgcn_readlane(take - at, k);
      for (unsigned long long left = choose_exact<T>(a, bh, qi, lane, nmay, need, mj, qs[wave]); left; left &= left - 1) {
        const int j = __builtin_amdgcn_readlane(mj, __ffsll(left) - 1);
        if (j >> 6 == lane) bits |= 1ull << (j & 63);
      }
    }
    int* const to = a.picked + ((long long)bh * a.nq + qi) * a.topk;
    int total;
    for (int c = places(bits, &total); bits; bits &= bits - 1) to[c++] = lane * 64 + __ffsll(bits) - 1;
    for (int t = total + lane; t < a.topk; t += 64) to[t] = -1;
  }
}

// ------------------------------------------------------------------------------------------------ attention
// Queries that pick their blocks one by one share no tile of keys.  Turned round they do: a workgroup takes ONE block (its keys in
// the registers of every wave, its values through LDS) and gathers the queries that picked it, 16 (query, head) rows to an MFMA
// tile -- S^T = K Q^T, softmax over the block, O^T = V^T P^T, where the S^T accumulators of two 16-key tiles are, after exp2, the B
// fragment of the second product -- and writes the block's result of each row with its maximum and sum; a second launch
// joins a row's blocks.  Keys are read once per block and range of queries instead of once per query; the price is that every (row,
// block) result passes through memory, which is what bounds the stage (2 (dv + 4) bytes written and read per row and block).
// Measured, lists / blocks / join: 16384 queries, 8 heads over 2, 16 blocks of 64 9.5 / 106 / 60 us (17 GMAC: 330 TFLOP/s; 270 MB of block
// results, read by the join at 4500 GB/s); 8 images x 1600 queries x 6 heads x 8 blocks 7 / 38 / 17 us.  The middle launch issues about 210
// vector instructions to a tile of 16 rows x 64 keys beside 18 MFMAs, 16 of them exponentials at a quarter of the rate (57 % of the SIMDs'
// cycles on the 128x128 map, the matrix pipe 15 %).  A tile of 16 neighbouring queries that read all the blocks any of them picked would
// do 2-5 times the work: 16 neighbours pick 76 of 256 blocks together there, 34 of 100 on the 80x80 map, 16 and 8 each.
//
// The softmax weights are rounded to the tensors' type (2^-8 of bf16, 2^-11 of fp16 at most) because the matrix pipe takes both factors in
// one type; their sum is that of the rounded ones.  With the block results below, the error against 64 bits is 2.2e-3 of the result in
// bf16, where rounding once alone makes 1.7e-3.
//
// A block's results pass unnormalised (sum of p v; the maximum and sum of p beside them in fp32).  For fp16 tensors they are fp32.  For
// bf16 tensors they are fp16 (off by 2^-11 at most, an eighth of a bf16 step; fp32 took 278 instead of 150 us on the 128x128 map):
// a power of two per unit, carried by the weights (exact in bf16), puts the unit's largest value at 2^8, so that the sums fill fp16's
// range from the top; the join scales back.  Where no readable value of the unit is under 2^-22 of the largest, the sum of p |v| is in
// fp16's normal range for every row and channel (the largest p is 1).  The results of other units -- zeros, channels of very different
// size, large values that may have next to no weight -- stay in fp32: the upper 16 bits where the others have their fp16, the lower 16
// bits in a second array that is touched for such units alone, and the rows' sums of p are stored as their negatives.  Values half of
// which are zeros: 334 instead of 184 us on the 128x128 map, 77 instead of 59 on the 40x40 maps (whole calls in a graph).  Looking at the
// results row by row instead costs registers that the loop over the tiles does not have (spills): 205 us on the 128x128 map for any values.
//
// Lists: 64 queries form a group; lists[group] holds its (query, slot) pairs sorted by block, starts[group][j] where block j's begin.
// A block of 128 keys is two units of 64 (two results per slot): one unit's fragments fill the registers.

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  typedef _Float16 part;  // a block's results between the launches
  // sums of weighted values are held times 2^-down: 64 keys x 64 blocks of the largest values stay in fp32's range
  static constexpr int down = 16;
  typedef bf16x8 t8;
  typedef bf16x4 t4;
  static __device__ __forceinline__ f32x4 mfma(t8 a, t8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Vec<_Float16> {
  typedef float part;
  static constexpr int down = 0;
  typedef f16x8 t8;
  typedef _Float16 t4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4 mfma(t8 a, t8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ unsigned pack(float lo, float hi) {  // (round to nearest even)
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, h2{(_Float16)lo, (_Float16)hi});
  }
};

struct AttendArgs {
  BlockArgs a;
  int subs, slots;          // units per block, results per row: topk * subs
  int groups, range, nrange;  // groups of 64 queries per image; groups of a workgroup's range; ranges
  unsigned short* starts;   // [batch * kv][groups][nb + 1]
  unsigned short* lists;    // [batch * kv][groups][64 * topk]: query (6 bits) << 6 | slot
  int g0, gn, cq;           // this launch's groups of queries [g0, g0 + gn), and how many queries `part` has room for
  long long mlrow;          // nq * group
  int q32;                  // offsets of q inside a range of queries fit 32 bits, its strides 24
  signed char* vexp;        // [b * kv + h][nb * subs]: bf16 tensors: a unit's results are times 2^vexp
  void* part;               // [row][slots][DVP], row = ((b * kv + h) * cq + i - 64 g0) * group + head in the group
  long long low;            // bf16 tensors: so many bytes behind `part` is the same again, for the lower halves of results in fp32
  float2* ml;               // [b * kv + h][slots][nq * group]: maximum (log2), sum (negative: the results are in fp32) -- rows together: a
                            // unit's neighbours share lines
};

// One wave per (image, kv head, 64 queries): the group's picks sorted by block.  A block counts once per query; slots that name no
// block, or one again, get a result of weight 0.
__global__ __launch_bounds__(64) void block_lists_kernel(AttendArgs p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char list_sm[];
  unsigned long long* word = reinterpret_cast<unsigned long long*>(list_sm);  // [nb]: which queries picked the block
  unsigned short* start = reinterpret_cast<unsigned short*>(word + p.a.nb);   // [nb + 1]
  const int lane = threadIdx.x, nb = p.a.nb, topk = p.a.topk;
  const int grp = blockIdx.x % p.groups, bh = blockIdx.x / p.groups;
  const int i = grp * 64 + lane;
  for (int j = lane; j < nb; j += 64) word[j] = 0;
  __syncthreads();
  const long long q = (long long)bh * p.a.nq + i;
  const int* pick = p.a.picked + q * topk;
  const unsigned long long me = 1ull << lane;
  unsigned long long first = 0;  // this query's slots that count
  constexpr int U = 8;           // picks in flight together (one by one a memory latency each: the launch took 11 instead of 9 us on the 128x128 map)
  auto picks = [&](int t0, int (&js)[U]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) js[u] = i < p.a.nq && t0 + u < topk ? pick[t0 + u] : -1;
  };
  for (int t0 = 0; t0 < topk; t0 += U) {
    int js[U];
    picks(t0, js);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = js[u];
      if (j >= 0 && j < nb && !(word[j] & me)) {  // (only this lane sets this bit)
        atomicOr(&word[j], me);
        first |= 1ull << (t0 + u);
      } else if (i < p.a.nq && t0 + u < topk) {
        for (int sub = 0; sub < p.subs; ++sub)
          for (int g = 0; g < p.a.group; ++g)
            p.ml[((long long)bh * p.slots + (t0 + u) * p.subs + sub) * p.mlrow + (long long)i * p.a.group + g] = float2{-__builtin_huge_valf(), 0.f};
      }
    }
  }
  __syncthreads();
  int base = 0;
  for (int j0 = 0; j0 < nb; j0 += 64) {  // where each block's queries begin
    const int j = j0 + lane;
    const int n = j < nb ? __popcll(word[j]) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (j < nb) start[j] = (unsigned short)(base + x - n);
    base += __shfl(x, 63);
  }
  if (lane == 0) start[nb] = (unsigned short)base;
  __syncthreads();
  const long long at = (long long)bh * p.groups + grp;
  unsigned short* list = p.lists + at * (64 * topk);
  for (int t0 = 0; t0 < topk; t0 += U) {
    int js[U];
    picks(t0, js);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first >> (t0 + u) & 1) list[start[js[u]] + __popcll(word[js[u]] & (me - 1))] = (unsigned short)(lane << 6 | (t0 + u));
  }
  for (int j = lane; j <= nb; j += 64) p.starts[at * (nb + 1) + j] = start[j];
}

// Where the values of channel c lie in LDS: keys in a row, the row's parts exchanged by xor with the channel -- lanes that write the
// same two keys of eight channels 8 apart would all meet in two banks.
template <int KEYS, int DVP>
__device__ __forceinline__ int value_at(int c, int key) {
  constexpr int STEP = DVP == 128 ? 8 : 16;  // keys that stay together
  return c * (KEYS + 8) + (key ^ (((c >> 4) & (KEYS / STEP - 1)) * STEP));
}

// DIRECT: one wave per (image, kv head, query, slot, unit) straight from `picked` -- few queries, where lists would hold one entry.
// Four workgroups on a CU where the fragments leave room (128 registers; at 131, three of them, the 128x128 map's launch took 119 instead
// of 108 us; five spill), three for wide values of bf16 tensors (2 x 6400 queries, 6 heads, key width 64, value width 128: 70 us; two 91).
template <typename T, int KEYS, int DK32, int DV16, bool DIRECT>
__global__ __launch_bounds__(DIRECT ? 64 : 256, DIRECT || DK32 > 2 ? 2 : DV16 == 4 ? 4 : sizeof(typename Vec<T>::part) == 2 ? 3 : 2) void block_attend_kernel(AttendArgs p) {
  typedef typename Vec<T>::t8 t8;
  typedef typename Vec<T>::t4 t4;
  constexpr int NT = DIRECT ? 64 : 256;
  typedef std::conditional_t<DIRECT, float, typename Vec<T>::part> part_t;  // (few rows: nothing to save)
  constexpr bool HALF = sizeof(part_t) == 2;
  constexpr int DOWN = Vec<T>::down;
  constexpr int KT = KEYS / 16, KS = KEYS / 32, DVP = DV16 * 16, VP = KEYS + 8;
  __shared__ __attribute__((aligned(16))) T sVt[DVP * VP];
  extern __shared__ unsigned rows[];  // [64 * range]: group in the range << 12 | query << 6 | slot
  __shared__ int first[DIRECT ? 1 : 65], from[DIRECT ? 1 : 64];  // per group of the range: its place in `rows`, in its list
  const BlockArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, n = lane & 15;
  const float ninf = -__builtin_huge_valf();
  // ---- which block
  int unit = xcd_remap((int)blockIdx.x, (int)gridDim.x);  // neighbours share an image, a head, a range of queries: one L2
  int sub = 0, j, bh, grp0 = 0, nrows, qdirect = 0, tdirect = 0;
  if (KEYS == 64) {
    sub = unit % p.subs;
    unit /= p.subs;
  }
  if constexpr (DIRECT) {
    tdirect = unit % a.topk;
    unit /= a.topk;
    qdirect = unit % a.nq;
    bh = unit / a.nq;
    const int* pick = a.picked + ((long long)bh * a.nq + qdirect) * a.topk;
    j = pick[tdirect];
    bool use = j >= 0 && j < a.nb;
    for (int t = 0; t < tdirect; ++t) use = use && pick[t] != j;
    if (!use) {
      const long long at = ((long long)bh * p.slots + tdirect * p.subs + sub) * p.mlrow + (long long)qdirect * a.group;
      for (int e = lane; e < a.group; e += 64) p.ml[at + e] = float2{ninf, 0.f};
      return;
    }
    nrows = a.group;
  } else {
    j = unit % a.nb;
    unit /= a.nb;
    grp0 = p.g0 + unit % p.nrange * p.range;
    bh = unit / p.nrange;
  }
  const int h = bh % a.kv, b = bh / a.kv;
  const int k0 = j * a.block + sub * KEYS;
  const int kn = min(min(KEYS, a.block - sub * KEYS), a.nk - k0);  // keys of this unit; <= 0: none
  const bool lok = lane < kn && (!a.mask || a.mask[b * a.mask_stride + k0 + lane]);
  const unsigned long long ok = __ballot(lok);  // the keys that may be read
  // ---- keys: fragments of the first product (row = key, 8 dims of group g).  Keys and values are asked for ahead of the lists.
  t8 kf[KT][DK32];
  const T* kb = static_cast<const T*>(a.k.p) + b * a.k.sb + h * a.k.sh;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int c = 0; c < DK32; ++c) {
      kf[t][c] = t8{};
      if (t * 16 + n < kn && (c * 4 + g) * 8 < a.dk) kf[t][c] = *reinterpret_cast<const t8*>(kb + token(a, k0 + t * 16 + n) * a.k.st + (c * 4 + g) * a.k.sc);
    }
  // ---- values; a masked one counts as 0 whatever it holds.  A thread moves two keys x 8 channels.
  __shared__ unsigned ends[NT / 64];  // of a wave's values: the largest, 0x7FFF - the smallest
  const T* vb = static_cast<const T*>(a.v.p) + b * a.v.sb + h * a.v.sh;
  constexpr int ITEMS = KEYS / 2 * (DVP / 8), NV = (ITEMS + NT - 1) / NT;
  u32x4 v[NV][2];
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int it = tid + x * NT, c8 = it % (DVP / 8), key = it / (DVP / 8) * 2;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      v[x][u] = u32x4{0, 0, 0, 0};
      if (it < ITEMS && c8 * 8 < a.dv && (ok >> (key + u) & 1))
        v[x][u] = *reinterpret_cast<const u32x4*>(vb + token(a, k0 + key + u) * a.v.st + c8 * a.v.sc);
    }
  }
  // ---- which queries
  if constexpr (!DIRECT) {
    const int ng = min(p.range, p.g0 + p.gn - grp0);
    if (wave == 0) {  // a lane per group: where its share of the list begins, here and there
      int lo = 0, cnt = 0;
      const long long at = (long long)bh * p.groups + grp0 + lane;
      if (lane < ng) {
        lo = p.starts[at * (a.nb + 1) + j];
        cnt = p.starts[at * (a.nb + 1) + j + 1] - lo;
      }
      int x = cnt;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      first[lane] = x - cnt;
      from[lane] = lo;
      if (lane == 63) first[64] = x;
    }
    __syncthreads();
    const int total = first[64];
    nrows = total * a.group;
    if (nrows == 0) return;
    for (int e = tid; e < total; e += NT) {  // the group that holds entry e: the last one that begins at or before it
      int x = 0;
#pragma unroll
      for (int o = 32; o; o >>= 1) x += first[x + o] <= e ? o : 0;
      const long long at = ((long long)bh * p.groups + grp0 + x) * (64 * a.topk);
      rows[e] = (unsigned)x << 12 | p.lists[at + from[x] + e - first[x]];
    }
  }
  // ... transposed, keys in a row
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int it = tid + x * NT, c8 = it % (DVP / 8), key = it / (DVP / 8) * 2;
    if (it < ITEMS)
#pragma unroll
      for (int e = 0; e < 8; ++e)  // (lower halves of a pair of words, upper halves)
        *reinterpret_cast<unsigned*>(sVt + value_at<KEYS, DVP>(c8 * 8 + e, key)) =
            __builtin_amdgcn_perm(v[x][1][e >> 1], v[x][0][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
  }
  // The power of two 2^up that puts the largest finite |v| at 2^8 (values under 2^-92: less): sums of 64 weighted values stay under 2^15.
  // (Results in fp32: at 2^100, or 2^up = 2^100.)
  // The weights carry it (as far as they can without leaving bf16's range; the rest, where values are beyond 2^60, the stores).
  float upw = HALF ? 0.f : -DOWN, ups = 1.f;
  bool spread = false;  // some readable value is under 2^-22 of the largest
  if constexpr (HALF) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 big = {0, 0}, small = {0, 0};
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int it = tid + x * NT, c8 = it % (DVP / 8), key = it / (DVP / 8) * 2;
        const bool there = it < ITEMS && c8 * 8 < a.dv && (ok >> (key + u) & 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          us2 m = __builtin_bit_cast(us2, v[x][u][e] & 0x7FFF7FFFu);
          small = __builtin_elementwise_max(small, there ? us2{0x7FFF, 0x7FFF} - m : us2{0, 0});
          m = us2{m[0] < 0x7F80 ? m[0] : (unsigned short)0, m[1] < 0x7F80 ? m[1] : (unsigned short)0};
          big = __builtin_elementwise_max(big, m);
        }
      }
    const unsigned both = wave_max2(__builtin_bit_cast(unsigned, __builtin_elementwise_max(us2{big[0], small[0]}, us2{big[1], small[1]})));
    if (lane == 0) ends[wave] = both;
    __syncthreads();
    us2 all = {0, 0};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) all = __builtin_elementwise_max(all, __builtin_bit_cast(us2, ends[w]));
    const unsigned ends2 = (unsigned)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, all));  // (the same in every lane)
    const unsigned vmax = ends2 & 0xFFFF, vmin = 0x7FFF - (ends2 >> 16);
    const int e = (int)(vmax >> 7) - 127, em = (int)(vmin >> 7);  // floor(log2 of the largest) (-127: zeros, or not normal); 0: a zero, or not normal
    int up = vmax ? min(8 - e, 100) : 0;
    spread = vmax != 0 && (em == 0 || em - 127 + up < -14);
    if (spread) up = min(100 - e, 100);
    const int uw = max(up, -60);
    upw = (float)uw;
    ups = __uint_as_float((unsigned)(up - uw + 127) << 23);  // (up - uw >= -59)
    if (tid == 0) p.vexp[((long long)bh * a.nb + j) * p.subs + sub] = (signed char)-up;
  } else {
    __syncthreads();
  }
  unsigned okt = 0;  // this lane's keys t * 16 + 4 g + r, four bits per tile
#pragma unroll
  for (int t = 0; t < KT; ++t) okt |= (unsigned)(ok >> (t * 16 + 4 * g) & 15) << (4 * t);
  // values: which channel is row i of tile d -- one that lets the four lanes of a query store 64 neighbouring bytes at a time
  auto channel = [](int d, int i) { return HALF ? (d >> 1) * 32 + (i >> 2) * 8 + (d & 1) * 4 + (i & 3) : d * 16 + i; };
  t8 vf[DV16][KS];
#pragma unroll
  for (int d = 0; d < DV16; ++d)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const t4 lo = *reinterpret_cast<const t4*>(sVt + value_at<KEYS, DVP>(channel(d, n), s * 32 + 4 * g));
      const t4 hi = *reinterpret_cast<const t4*>(sVt + value_at<KEYS, DVP>(channel(d, n), s * 32 + 16 + 4 * g));
      vf[d][s] = t8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  // scores are scaled by |scale| inside the exponential's fma; a negative scale flips the queries' signs
  const float scale = fabsf(a.scale) * 1.44269504088896340736f;
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
  const bool all = ok == ~0ull >> (64 - KEYS);  // no key is masked: uniform
  const float downw = __builtin_amdgcn_exp2f(-upw);  // (a whole power: exact; 1 for fp16 tensors)
  t8 one;
#pragma unroll
  for (int e = 0; e < 8; ++e) one[e] = (T)1.f;

  // a tile's queries: lane column n is (query, head) row f.  q0: the first query that this unit may have; everything per row is a
  // 24-bit product from there (a full 32-bit one takes four times as long)
  struct Row {
    int q, head, slot;  // query behind q0
    bool live;
    t8 f[DK32];
  };
  const int q0 = DIRECT ? qdirect : grp0 * 64;
  const T* const qb = head_ptr<const T>(a, a.q, b, q0, h * a.group);
  const int qtok = token(a, q0);
  part_t* const pb = static_cast<part_t*>(p.part) + ((long long)bh * p.cq + (q0 - p.g0 * 64)) * a.group * p.slots * DVP;
  float2* const mlb = p.ml + (long long)bh * p.slots * p.mlrow + (long long)q0 * a.group;
  auto fetch = [&](int tile, Row& w) __attribute__((always_inline)) {
    const int f = tile * 16 + n;
    w.live = f < nrows;
    const int fc = w.live ? f : 0;
    int e = fc;
    w.head = 0;
    if (a.group > 1) {
      e = (int)__umulhi((unsigned)fc, a.magic);
      w.head = fc - __mul24(e, a.group);
    }
    if constexpr (DIRECT) {
      w.q = 0;
      w.slot = tdirect * p.subs + sub;
    } else {
      const unsigned x = rows[e];
      w.q = (int)(x >> 6);
      w.slot = __mul24((int)(x & 63), p.subs) + sub;
    }
    const T* qp;
    if (a.W)
      qp = qb + (token(a, q0 + w.q) - qtok) * a.q.st + w.head * a.q.sh;
    else if (p.q32)
      qp = qb + (unsigned)(__umul24((unsigned)w.q, (unsigned)a.q.st) + __umul24((unsigned)w.head, (unsigned)a.q.sh));
    else
      qp = qb + w.q * a.q.st + w.head * a.q.sh;
#pragma unroll
    for (int c = 0; c < DK32; ++c) {
      w.f[c] = t8{};
      if ((c * 4 + g) * 8 < a.dk) w.f[c] = *reinterpret_cast<const t8*>(qp + (c * 4 + g) * a.q.sc);
    }
  };
  const int ntiles = (nrows + 15) >> 4;
  constexpr int NW = NT / 64;
  Row next;
  if (wave < ntiles) fetch(wave, next);
  for (int tile = wave; tile < ntiles; tile += NW) {
    Row w = next;
    if (tile + NW < ntiles) fetch(tile + NW, next);
    if (flip)
#pragma unroll
      for (int c = 0; c < DK32; ++c) {
        u32x4 x = __builtin_bit_cast(u32x4, w.f[c]);
#pragma unroll
        for (int d = 0; d < 4; ++d) x[d] ^= flip;
        w.f[c] = __builtin_bit_cast(t8, x);
      }
    f32x4 s[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DK32; ++c) s[t] = Vec<T>::mfma(kf[t][c], w.f[c], s[t]);
    }
    float m = ninf;
    u32x4 pw[KS];
    if (all) {
      // max(x, y) = med3(x, y, inf): one instruction where fmaxf first quiets a possible signalling NaN (a NaN score makes NaN below)
      float mt[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {  // (pairs, then pairs of pairs: a short chain)
        const float x = __builtin_amdgcn_fmed3f(s[t][0], s[t][1], __builtin_huge_valf());
        mt[t] = __builtin_amdgcn_fmed3f(x, __builtin_amdgcn_fmed3f(s[t][2], s[t][3], __builtin_huge_valf()), __builtin_huge_valf());
      }
#pragma unroll
      for (int t = 1; t < KT; ++t) mt[0] = __builtin_amdgcn_fmed3f(mt[0], mt[t], __builtin_huge_valf());
      m = quad_max(mt[0]) * scale;
      const float base = (m == ninf ? 0.f : m) - upw;  // (every score -inf: all weights 0)
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
          pw[t >> 1][(t & 1) * 2 + r / 2] = Vec<T>::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale, -base)),
                                                         __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + 1], scale, -base)));
    } else {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = okt >> (4 * t + r) & 1 ? fmaxf(m, s[t][r]) : m;
      m = quad_max(m);
      m = m == ninf ? m : m * scale;  // (no key: -inf, also where the scale is 0)
      const float base = (m == ninf ? 0.f : m) - upw;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale, -base)), e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + 1], scale, -base));
          pw[t >> 1][(t & 1) * 2 + r / 2] = Vec<T>::pack(okt >> (4 * t + r) & 1 ? e0 : 0.f, okt >> (4 * t + r + 1) & 1 ? e1 : 0.f);
        }
    }
    t8 pf[KS];
#pragma unroll
    for (int x = 0; x < KS; ++x) pf[x] = __builtin_bit_cast(t8, pw[x]);
    // the weights' sum by the matrix pipe too: a row of ones; every lane of a query gets it, and it is the sum of what multiplies v
    f32x4 lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < KS; ++x) lsum = Vec<T>::mfma(one, pf[x], lsum);
    const float l = DOWN ? lsum[0] * downw : lsum[0];
    f32x4 o[DV16];
#pragma unroll
    for (int d = 0; d < DV16; ++d) {
      o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) o[d] = Vec<T>::mfma(vf[d][x], pf[x], o[d]);
    }
    if (!w.live) continue;
    const unsigned local = __umul24((unsigned)w.q, (unsigned)a.group) + (unsigned)w.head;  // row behind q0's first: below 4096 * 1000
    part_t* const dst = pb + (long long)(__umul24(local, (unsigned)p.slots) + (unsigned)w.slot) * DVP;
    if constexpr (HALF) {
      if (ups != 1.f)
#pragma unroll
        for (int d = 0; d < DV16; ++d) o[d] *= ups;
      auto pk = [](float lo, float hi) {  // (round to nearest even)
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{lo, hi}), h2));
      };
      if (!spread) {
#pragma unroll
        for (int d = 0; d < DV16; d += 2)
          *reinterpret_cast<u32x4*>(dst + channel(d, 4 * g)) =
              u32x4{pk(o[d][0], o[d][1]), pk(o[d][2], o[d][3]), pk(o[d + 1][0], o[d + 1][1]), pk(o[d + 1][2], o[d + 1][3])};
      } else {
        auto halves = [](float x, float y, unsigned which) { return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), which); };
#pragma unroll
        for (int d = 0; d < DV16; d += 2)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const unsigned which = u ? 0x05040100u : 0x07060302u;  // upper halves to part, lower ones behind it
            *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(dst + channel(d, 4 * g)) + (u ? p.low : 0)) =
                u32x4{halves(o[d][0], o[d][1], which), halves(o[d][2], o[d][3], which), halves(o[d + 1][0], o[d + 1][1], which),
                      halves(o[d + 1][2], o[d + 1][3], which)};
          }
      }
    } else {
#pragma unroll
      for (int d = 0; d < DV16; ++d) *reinterpret_cast<f32x4*>(dst + channel(d, 4 * g)) = o[d];
    }
    if (g == 0) mlb[(long long)w.slot * p.mlrow + local] = float2{m, spread ? -l : l};
  }
}

// out = the slots' results weighted by their sums; one thread per (row, 8 channels)
template <typename T, typename P, int DVP>
__global__ __launch_bounds__(256) void block_join_kernel(AttendArgs p) {
  typedef typename Vec<T>::t8 t8;
  const BlockArgs& a = p.a;
  constexpr int C = DVP / 8;
  const int c = (int)(threadIdx.x % C) * 8;
  const unsigned prow = blockIdx.x * (256 / C) + threadIdx.x / C;  // rows of this launch's queries, fewer than 2^31
  const unsigned cq = (unsigned)min(p.gn * 64, a.nq - p.g0 * 64);
  if (prow >= (unsigned)a.batch * (unsigned)a.heads * cq || c >= a.dv) return;
  const unsigned e = prow / (unsigned)a.group, q = e / cq;
  const int gh = (int)(prow - e * (unsigned)a.group), i = p.g0 * 64 + (int)(e - q * cq), bh = (int)q;
  const float2* ml = p.ml + (long long)bh * p.slots * p.mlrow + (long long)i * a.group + gh;
  typedef P p8 __attribute__((ext_vector_type(8)));
  constexpr bool HALF = sizeof(P) == 2;
  const int* pick = a.picked + ((long long)bh * a.nq + i) * a.topk;
  const P* part = static_cast<const P*>(p.part) + (((long long)bh * p.cq + i - p.g0 * 64) * a.group + gh) * p.slots * DVP + c;
  constexpr int U = 8;  // slots whose loads are in flight together
  float m = -__builtin_huge_valf();
  for (int t0 = 0; t0 < p.slots; t0 += U) {
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = ml[min(t0 + u, p.slots - 1) * p.mlrow].x;
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(m, x[u]);
  }
  const float base = m == -__builtin_huge_valf() ? 0.f : m;
  float acc[8] = {}, sum = 0.f;
  for (int t0 = 0; t0 < p.slots; t0 += U) {
    float w[U], l[U];
    int ve[U];
    p8 y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(t0 + u, p.slots - 1);
      const float2 x = ml[t * p.mlrow];
      y[u] = *reinterpret_cast<const p8*>(part + t * DVP);  // (whatever lies there where the slot has no block: not used)
      ve[u] = 0;
      if constexpr (HALF) {
        const int j = pick[p.subs == 2 ? t >> 1 : t];
        ve[u] = p.vexp[((long long)bh * a.nb + (j >= 0 && j < a.nb ? j : 0)) * p.subs + (p.subs == 2 ? t & 1 : 0)];
      }
      w[u] = __builtin_amdgcn_exp2f(x.x - base);
      l[u] = t0 + u < p.slots ? x.y : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (l[u] == 0.f) continue;
      sum += w[u] * fabsf(l[u]);
      const float x = HALF ? __builtin_amdgcn_ldexpf(w[u], ve[u] - Vec<T>::down) : w[u];
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)y[u][e];
      if constexpr (HALF) {
        if (l[u] < 0.f) {  // in fp32, as two halves
          typedef unsigned short us8 __attribute__((ext_vector_type(8)));
          const us8 hi = __builtin_bit_cast(us8, y[u]), lo = *reinterpret_cast<const us8*>(reinterpret_cast<const char*>(part + (t0 + u) * DVP) + p.low);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = __uint_as_float((unsigned)hi[e] << 16 | lo[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += x * f[e];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  t8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (T)(acc[e] * inv * (float)(1 << Vec<T>::down));
  *reinterpret_cast<t8*>(head_ptr<T>(a, a.o, bh / a.kv, i, bh % a.kv * a.group + gh) + (c >> 3) * a.o.sc) = y;
}

// Few queries and blocks: one workgroup per (image, kv head, query, 16 query heads), a wave per slot and unit in turn with the running
// maximum and sum of its softmax, joined through LDS -- one launch, no workspace.  Bound by the latency of a round (block read, transposed,
// multiplied: 3-5 us) and by launches; 64 queries of width 128, 268 MB of blocks: 53 us, 5000 GB/s.
template <typename T, int KEYS, int DK32, int DV16>
__global__ __launch_bounds__(512, DK32 <= 2 && DV16 == 4 ? 4 : 2) void block_attend_few_kernel(AttendArgs p) {
  typedef typename Vec<T>::t8 t8;
  typedef typename Vec<T>::t4 t4;
  constexpr int KT = KEYS / 16, KS = KEYS / 32, DVP = DV16 * 16, VP = KEYS + 8;
  constexpr int REGION = DVP * VP * 2;  // bytes of LDS of a wave: its values, then its result: 16 rows of DVP floats, maximum and sum
  static_assert(REGION >= 64 * DVP + 128, "a wave's result takes the place of its values");
  extern __shared__ __attribute__((aligned(16))) unsigned char few_sm[];
  const BlockArgs& a = p.a;
  const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), nw = (int)blockDim.x >> 6;
  const float ninf = -__builtin_huge_valf();
  const int gt = (a.group + 15) >> 4;
  unsigned unit = blockIdx.x;
  const int tile = (int)(unit % (unsigned)gt);
  unit /= (unsigned)gt;
  const int i = (int)(unit % (unsigned)a.nq), bh = (int)(unit / (unsigned)a.nq), h = bh % a.kv, b = bh / a.kv;
  const int h0 = h * a.group + tile * 16, rows = min(16, a.group - tile * 16);
  T* const sVt = reinterpret_cast<T*>(few_sm + wave * REGION);
  const int* pick = a.picked + ((long long)bh * a.nq + i) * a.topk;
  const float scale = fabsf(a.scale) * 1.44269504088896340736f;
  const unsigned flip = a.scale < 0.f ? 0x80008000u : 0u;
  t8 qf[DK32];
#pragma unroll
  for (int c = 0; c < DK32; ++c) {
    u32x4 x = {0, 0, 0, 0};
    if ((c * 4 + g) * 8 < a.dk) x = *reinterpret_cast<const u32x4*>(head_ptr<const T>(a, a.q, b, i, h0 + min(n, rows - 1)) + (c * 4 + g) * a.q.sc);
#pragma unroll
    for (int d = 0; d < 4; ++d) x[d] ^= flip;
    qf[c] = __builtin_bit_cast(t8, x);
  }
  const T* kb = static_cast<const T*>(a.k.p) + b * a.k.sb + h * a.k.sh;
  const T* vb = static_cast<const T*>(a.v.p) + b * a.v.sb + h * a.v.sh;
  t8 one;
#pragma unroll
  for (int e = 0; e < 8; ++e) one[e] = (T)1.f;
  float m = ninf;
  f32x4 l = {0.f, 0.f, 0.f, 0.f}, o[DV16];
#pragma unroll
  for (int d = 0; d < DV16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int slot = wave; slot < p.slots; slot += nw) {
    const int t = p.subs == 2 ? slot >> 1 : slot, sub = p.subs == 2 ? slot & 1 : 0;
    const int j = pick[t];
    bool use = j >= 0 && j < a.nb;
    for (int u = 0; u < t; ++u) use = use && pick[u] != j;
    const int k0 = j * a.block + sub * KEYS, kn = min(min(KEYS, a.block - sub * KEYS), a.nk - k0);
    if (!use || kn <= 0) continue;  // (the same in every lane; no barrier of the workgroup in here)
    const bool lok = lane < kn && (!a.mask || a.mask[b * a.mask_stride + k0 + lane]);
    const unsigned long long ok = __ballot(lok);
    t8 kf[KT][DK32];
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int c = 0; c < DK32; ++c) {
        kf[x][c] = t8{};
        if (x * 16 + n < kn && (c * 4 + g) * 8 < a.dk) kf[x][c] = *reinterpret_cast<const t8*>(kb + token(a, k0 + x * 16 + n) * a.k.st + (c * 4 + g) * a.k.sc);
      }
    // values: two keys x 8 channels at a time, transposed into LDS
    constexpr int NV = KEYS / 2 * (DVP / 8) / 64;
#pragma unroll
    for (int x0 = 0; x0 < NV; x0 += 4) {
      u32x4 v[4][2];
#pragma unroll
      for (int x = 0; x < 4 && x0 + x < NV; ++x) {
        const int it = lane + (x0 + x) * 64, c8 = it % (DVP / 8), key = it / (DVP / 8) * 2;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          v[x][u] = u32x4{0, 0, 0, 0};
          if (c8 * 8 < a.dv && (ok >> (key + u) & 1)) v[x][u] = *reinterpret_cast<const u32x4*>(vb + token(a, k0 + key + u) * a.v.st + c8 * a.v.sc);
        }
      }
#pragma unroll
      for (int x = 0; x < 4 && x0 + x < NV; ++x) {
        const int it = lane + (x0 + x) * 64, c8 = it % (DVP / 8), key = it / (DVP / 8) * 2;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<unsigned*>(sVt + value_at<KEYS, DVP>(c8 * 8 + e, key)) =
              __builtin_amdgcn_perm(v[x][1][e >> 1], v[x][0][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
      }
    }
    f32x4 s[KT];
#pragma unroll
    for (int x = 0; x < KT; ++x) {
      s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DK32; ++c) s[x] = Vec<T>::mfma(kf[x][c], qf[c], s[x]);
    }
    unsigned okt = 0;  // this lane's keys x * 16 + 4 g + r, four bits per tile
#pragma unroll
    for (int x = 0; x < KT; ++x) okt |= (unsigned)(ok >> (x * 16 + 4 * g) & 15) << (4 * x);
    float top = ninf;
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = okt >> (4 * x + r) & 1 ? fmaxf(top, s[x][r]) : top;
    top = quad_max(top);
    top = top == ninf ? top : top * scale;  // (no key: -inf, also where the scale is 0)
    const float now = fmaxf(m, top), base = now == ninf ? 0.f : now;
    const float fade = __builtin_amdgcn_exp2f(m - base);
    m = now;
    u32x4 pw[KS];
#pragma unroll
    for (int x = 0; x < KT; ++x)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {  // (times 2^-down, which the division by their sum takes out again)
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], scale, -base - Vec<T>::down));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r + 1], scale, -base - Vec<T>::down));
        pw[x >> 1][(x & 1) * 2 + r / 2] = Vec<T>::pack(okt >> (4 * x + r) & 1 ? e0 : 0.f, okt >> (4 * x + r + 1) & 1 ? e1 : 0.f);
      }
    // (a wave's LDS accesses are carried out in order: its own writes are there)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    l *= fade;
#pragma unroll
    for (int x = 0; x < KS; ++x) l = Vec<T>::mfma(one, __builtin_bit_cast(t8, pw[x]), l);
#pragma unroll
    for (int d = 0; d < DV16; ++d) {
      o[d] *= fade;
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const t4 lo = *reinterpret_cast<const t4*>(sVt + value_at<KEYS, DVP>(d * 16 + n, x * 32 + 4 * g));
        const t4 hi = *reinterpret_cast<const t4*>(sVt + value_at<KEYS, DVP>(d * 16 + n, x * 32 + 16 + 4 * g));
        o[d] = Vec<T>::mfma(t8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, __builtin_bit_cast(t8, pw[x]), o[d]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the next values come behind these reads)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  // ---- join: row n's channels 16 d + 4 g + r of every wave
  float* const res = reinterpret_cast<float*>(sVt);
#pragma unroll
  for (int d = 0; d < DV16; ++d) *reinterpret_cast<f32x4*>(res + n * DVP + d * 16 + 4 * g) = o[d];
  if (g == 0) *reinterpret_cast<float2*>(res + 16 * DVP + 2 * n) = float2{m, l[0]};
  __syncthreads();
  for (int item = threadIdx.x; item < rows * (DVP / 8); item += (int)blockDim.x) {
    const int row = item / (DVP / 8), c = item % (DVP / 8) * 8;
    if (c >= a.dv) continue;
    float big = ninf;
    for (int w = 0; w < nw; ++w) big = fmaxf(big, reinterpret_cast<const float*>(few_sm + w * REGION)[16 * DVP + 2 * row]);
    const float base = big == ninf ? 0.f : big;
    float sum = 0.f, acc[8] = {};
    for (int w = 0; w < nw; ++w) {
      const float* r = reinterpret_cast<const float*>(few_sm + w * REGION);
      const float x = __builtin_amdgcn_exp2f(r[16 * DVP + 2 * row] - base), lw = r[16 * DVP + 2 * row + 1];
      if (lw == 0.f) continue;
      sum += x * lw;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += x * r[row * DVP + c + e];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    t8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (T)(acc[e] * inv);
    *reinterpret_cast<t8*>(head_ptr<T>(a, a.o, b, i, h0 + row) + (c >> 3) * a.o.sc) = y;
  }
}

// ------------------------------------------------------------------------------------------------ host
static long long round256(long long n) { return (n + 255) / 256 * 256; }

// a * b * c below 2^31 (factors below 2^31: a product in 64 bits could wrap around)
static bool fits31(long long a, long long b, long long c) { return (double)a * (double)b * (double)c < 2147483648.0; }

// A launch has fewer than 2^32 threads: a larger one is cut off, without an error.
static bool fits_grid(long long workgroups, int threads) { return workgroups * threads < 1LL << 32; }

static int check_heads(const std::string& who, const char* name, const yl_heads* t) {
  if (!t || !t->data) return fail(-1, who + ": null " + name);
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) || ((t->batch | t->token | t->head) & 7))
    return fail(-1, who + ": " + name + " must be 16-byte aligned with strides that are multiples of 8 elements");
  if (t->batch < 0 || t->token < 0 || t->head < 0) return fail(-1, who + ": " + name + " has a negative stride");
  return 0;
}

static void fill_errors(BlockArgs* a) {  // (block_score_kernel says what these are)
  a->part_err = (float)(((a->group > 1 ? 2 : 1) + 0.05) / (1 << 17));
  a->head_err = (float)((a->group - 1) * std::sqrt((double)a->group) * 1.01 / (1 << 24));  // (1.01: the norm is an fp32 sum too)
}

// sizes that the calls share -> BlockArgs; nothing is launched where batch * nq is 0
static int fill_args(const std::string& who, const yl_heads* q, const yl_heads* k, int dtype, int batch, int nq, int nk, int heads,
                     int kv_heads, int dk, int block, int topk, const uint8_t* mask, int64_t mask_stride, BlockArgs* a) {
  if (dtype != YL_BF16 && dtype != YL_F16) return fail(-1, who + ": bf16 or fp16 tensors");
  if (batch < 0 || nq < 0 || nk < 0) return fail(-1, who + ": a negative size");
  if (heads < 1 || kv_heads < 1 || heads % kv_heads) return fail(-1, who + ": the query heads must be a multiple of the kv heads");
  if (heads / kv_heads > 1000) return fail(-3, who + ": more than 1000 query heads to a kv head");
  if (dk < 8 || dk > 128 || dk % 8) return fail(-3, who + ": key widths are multiples of 8 up to 128");
  if (block != 32 && block != 64 && block != 128) return fail(-3, who + ": blocks of 32, 64 or 128 keys");
  if (topk < 1 || topk > BA_MAX_TOPK) return fail(-3, who + ": 1 to 64 blocks for a query");
  const long long nb = ((long long)nk + block - 1) / block;
  if (nb > BA_MAX_BLOCKS) return fail(-3, who + ": more than 4096 key blocks");
  if (!fits31(batch, heads, nq) || !fits31(batch, kv_heads, nb))
    return fail(-3, who + ": more rows or blocks than one launch covers");
  if (batch * (long long)nq == 0) return 0;
  if (int rc = check_heads(who, "q", q)) return rc;
  if (nk > 0)
    if (int rc = check_heads(who, "k", k)) return rc;
  if (mask && batch > 1 && mask_stride < nk) return fail(-1, who + ": the mask's row stride is smaller than a row");
  a->q = Heads{q->data, q->batch, q->token, q->head, 8};
  if (nk > 0) a->k = Heads{k->data, k->batch, k->token, k->head, 8};
  a->batch = batch, a->nq = nq, a->nk = nk, a->heads = heads, a->kv = kv_heads, a->group = heads / kv_heads;
  a->magic = (unsigned)((1ULL << 32) / a->group + 1);
  fill_errors(a);
  a->dk = dk, a->block = block, a->nb = (int)nb, a->topk = topk, a->mask = mask, a->mask_stride = mask_stride;
  return 0;
}

template <typename F>
static int by_type16(int dtype, F f) {
  if (dtype == YL_BF16) return f((__bf16*)nullptr);
  return f((_Float16*)nullptr);
}
#define BA_T(t) std::remove_pointer_t<decltype(t)>

}  // namespace yl

using namespace yl;

// ---- how the selection runs, and where things lie in the workspace
struct SelectPlan {
  long long mean, score, split, norm, count, all;  // byte offsets
};
static SelectPlan plan_select(BlockArgs* a) {
  SelectPlan p{};
  a->nbp = (a->nb + 15) / 16 * 16, a->dkp = (a->dk + 31) / 32 * 32;
  const long long bh = (long long)a->batch * a->kv;
  const bool few = a->nq <= SCORE_MAX_NQ;
  long long at = 0;
  auto take = [&](long long n) {
    const long long o = at;
    at += round256(n);
    return o;
  };
  p.mean = take(few ? 0 : 8 * bh * a->nb * a->dk);
  p.score = take(few ? 8 * bh * a->nq * a->nb : 0);
  p.split = take(few ? 0 : 4 * bh * a->nbp * a->dkp);
  p.norm = take(few ? 0 : 4 * bh * a->nb);
  p.count = take(4LL * a->batch * a->nb);
  p.all = at;
  return p;
}

// (block_mean_kernel; what score_by_size and select_run launch where there are many)
static int check_select(const BlockArgs& a) {
  const long long bh = (long long)a.batch * a.kv;
  const bool few = a.nq <= SCORE_MAX_NQ;
  const bool fits = fits_grid((bh * a.nb + 3) / 4, 256) &&
                    (few ? fits_grid(bh * a.nq, a.nb <= 256 ? 64 : a.nb <= 1024 ? 256 : 1024)
                         : fits_grid(bh * ((a.nq + 15) / 16) + 4, a.nb <= 256 ? 64 : a.nb <= 512 ? 256 : 512));
  return fits ? 0 : fail(-3, "block_select: more queries or blocks than one launch covers");
}

extern "C" int64_t yl_block_select_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dk, int block) {
  BlockArgs a{};
  yl_heads dummy{reinterpret_cast<void*>(16), 0, 0, 0};
  if (fill_args("block_select", &dummy, &dummy, YL_BF16, batch, nq, nk, heads, kv_heads, dk, block, 1, nullptr, 0, &a)) return -1;
  if (batch * (long long)nq == 0) return 0;
  return check_select(a) ? -1 : plan_select(&a).all;
}

template <typename T, bool SCORE, bool SMALL = false>
static int mean_launch(const BlockArgs& a, hipStream_t s) {
  const long long wg = ((long long)a.batch * a.kv * a.nb + 3) / 4;
  const int c = a.dk / 8, nw = std::max(SCORE_MAX_NQ, a.nb);
#define BA_MEAN(CP)                                                                                                           \
  do {                                                                                                                        \
    if constexpr (SMALL) hipLaunchKernelGGL((block_select_small_kernel<T, CP>), dim3(a.batch * a.kv), dim3(64 * nw), 0, s, a);   \
    else hipLaunchKernelGGL((block_mean_kernel<T, CP, SCORE>), dim3((unsigned)wg), dim3(256), 0, s, a);                           \
  } while (0)
  if (c <= 1) BA_MEAN(1);
  else if (c <= 2) BA_MEAN(2);
  else if (c <= 4) BA_MEAN(4);
  else if (c <= 8) BA_MEAN(8);
  else BA_MEAN(16);
#undef BA_MEAN
  YL_HIP(hipGetLastError());
  return 0;
}

template <typename T, int NW, int NT>
static int score_launch(const BlockArgs& a, int qtiles, unsigned units, hipStream_t s) {
  if constexpr (NW > 1)
    hipLaunchKernelGGL((block_score_wide_kernel<T, NW, NT>), dim3(units), dim3(64 * NW), 0, s, a, qtiles);
  else
    hipLaunchKernelGGL((block_score_kernel<T, NT>), dim3((units + 3) / 4), dim3(256), 0, s, a, qtiles);
  YL_HIP(hipGetLastError());
  return 0;
}
// One wave per 16 queries up to 128 blocks (6400 of them: 38 us where four waves take 100, the whole call).  Above, as few waves as have
// the registers where 16-query tiles alone fill the card (256 blocks, 8192 tiles: one wave 102, four 140 us; 512 blocks, 4096 tiles: four
// 145, eight 167 us), more waves where they do not (256 blocks, 512 tiles: 33 and 27 us; 512 blocks, 128 tiles: 31 and 28 us).
template <typename T>
static int score_by_size(const BlockArgs& a, hipStream_t s) {
  const int qtiles = (a.nq + 15) / 16;
  const unsigned units = (unsigned)((long long)a.batch * a.kv * qtiles);  // (below 2^31)
  if (a.nb <= 64) return score_launch<T, 1, 4>(a, qtiles, units, s);
  if (a.nb <= 128) return score_launch<T, 1, 8>(a, qtiles, units, s);
  if (a.nb <= 256) return units < 2048 ? score_launch<T, 4, 4>(a, qtiles, units, s) : score_launch<T, 1, 16>(a, qtiles, units, s);
  if (a.nb <= 512) return units <= 512 ? score_launch<T, 8, 4>(a, qtiles, units, s) : score_launch<T, 4, 8>(a, qtiles, units, s);
  if (a.nb <= 1024) return score_launch<T, 8, 8>(a, qtiles, units, s);
  return a.nb <= 2048 ? score_launch<T, 8, 16>(a, qtiles, units, s) : score_launch<T, 8, 32>(a, qtiles, units, s);
}

// the selection of `a` (sizes and tensors filled in) into a.picked, with plan `p` and its workspace
static int select_run(BlockArgs& a, const SelectPlan& p, int dtype, char* w, hipStream_t s) {
  a.mean = reinterpret_cast<double*>(w + p.mean), a.score = reinterpret_cast<double*>(w + p.score);
  a.split = reinterpret_cast<__bf16*>(w + p.split), a.norm = reinterpret_cast<float*>(w + p.norm);
  a.count = reinterpret_cast<int*>(w + p.count);
  return by_type16(dtype, [&](auto* t) {
    typedef BA_T(t) T;
    const bool few = a.nq <= SCORE_MAX_NQ;
    if (few && a.nb <= SMALL_BLOCKS && std::min(a.block, a.nk) * a.dk <= SMALL_BLOCK &&
        fits_grid((long long)a.batch * a.kv, 64 * std::max(SCORE_MAX_NQ, a.nb)))
      return mean_launch<T, true, true>(a, s);
    if (a.nb > 0)
      if (int rc = few ? mean_launch<T, true>(a, s) : mean_launch<T, false>(a, s)) return rc;
    if (!few && a.nb > 0) return score_by_size<T>(a, s);
    const dim3 grid((unsigned)(a.batch * a.kv * a.nq));
    if (a.nb <= 256) hipLaunchKernelGGL(block_select_kernel<1>, grid, dim3(64), 0, s, a);
    else if (a.nb <= 1024) hipLaunchKernelGGL(block_select_kernel<4>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(block_select_kernel<16>, grid, dim3(1024), 0, s, a);
    YL_HIP(hipGetLastError());
    return 0;
  });
}

extern "C" int yl_block_select(const yl_heads* q, const yl_heads* k, int dtype, int batch, int nq, int nk, int heads, int kv_heads,
                               int dk, int block, int topk, const uint8_t* mask, int64_t mask_stride, int32_t* picked, void* work,
                               int64_t work_bytes, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  BlockArgs a{};
  if (int rc = fill_args("block_select", q, k, dtype, batch, nq, nk, heads, kv_heads, dk, block, topk, mask, mask_stride, &a)) return rc;
  if (batch * (long long)nq == 0) return 0;
  if (!picked) return fail(-1, "block_select: null pointer");
  if (int rc = check_select(a)) return rc;
  const SelectPlan p = plan_select(&a);
  if (p.all > 0 && (!work || work_bytes < p.all || (reinterpret_cast<uintptr_t>(work) & 15)))
    return fail(-1, "block_select: workspace missing, too small or not 16-byte aligned");
  a.picked = picked;
  return select_run(a, p, dtype, static_cast<char*>(work), s);
}

// ---- how the attention runs: sizes, and where things lie in the workspace
struct AttendPlan {
  bool direct, few;
  int subs, slots, groups, range, dvp;
  int chunk;               // groups of queries whose block results are in memory together
  long long starts, lists, vexp, part, low, ml, all;  // byte offsets
};

// block results in memory at once, the second array of bf16 tensors apart (measured: 128 MB and more the same time, 64 MB 15 % more, 16 MB twice)
constexpr long long CHUNK_BYTES = 256LL << 20;
static AttendPlan plan_attend(const BlockArgs& a, int dv, int dtype) {
  AttendPlan p{};
  p.subs = a.block == 128 ? 2 : 1;
  p.slots = a.topk * p.subs;
  p.dvp = dv <= 64 ? 64 : 128;
  p.groups = (a.nq + 63) / 64;
  // the lists pay where a block is picked often; below that, a wave per (query, block)
  p.direct = a.nq <= 4 || (long long)a.nq * a.topk <= 2LL * a.nb;
  // One launch for one or two rounds of eight waves.  One query, 8 kv heads, blocks of 64, that launch / two launches (captured, us):
  // width 64, 8 blocks 8.1 / 8.5, 16 blocks 10.9 / 10.1, 32 blocks 17.6 / 13.7; width 128, 8 blocks 12.2 / 10.3, 16 blocks 17.9 / 12.2;
  // a call of its own is 3 us less for the host.  With many queries it wins further (32 images, width 128, 16 blocks 26 / 32; 16 images with
  // 4 query heads to one 20 / 22), but for 2048 workgroups of one round (55 / 47).
  const long long wgs = (long long)a.batch * a.kv * a.nq * ((a.group + 15) / 16);
  const int work = std::min(a.topk, std::max(1, a.nb)) * p.subs;  // slots that can name a block of their own
  // ... and in place of the lists where queries times blocks are so few that sharing keys saves less than the launches cost (one launch /
  // lists, call): 400 queries x 2 heads x 4 blocks 11.2 / 19.7, 64 x 8 x 16 18.6 / 22.8, 128 x 8 x 8 20.5 / 19.1; 256 queries, 32 heads over 2,
  // 8 blocks 11.7 / 28.4; width 128: 32 x 8 x 8 15.8 / 16.1, 64 x 8 x 16 38.6 / 35.2.
  p.few = (p.direct || wgs * work * p.dvp <= 1 << 19) && (work * p.dvp <= 1024 || (work <= 16 && wgs >= 128));
  p.direct = p.direct || p.few;
  if (p.few) return p;  // (one launch, no workspace)
  // a workgroup's range of queries: about 512 (query, head) rows, 32 tiles, for an average block
  const long long per64 = 64LL * a.topk * a.group;
  p.range = (int)std::min<long long>(64, std::max<long long>(1, 512LL * std::max(1, a.nb) / per64));
  const long long rows = (long long)a.batch * a.nq * a.heads, bg = (long long)a.batch * a.kv * p.groups;
  const int part_bytes = dtype == YL_BF16 && !p.direct ? 2 : 4;
  p.chunk = p.groups;
  if (!p.direct) {
    const long long group_bytes = (long long)part_bytes * a.batch * a.heads * 64 * p.slots * p.dvp;
    p.chunk = (int)std::min<long long>(p.groups, std::max<long long>(1, CHUNK_BYTES / group_bytes));
  }
  p.range = std::min(p.range, p.chunk);
  long long at = 0;
  auto take = [&](long long n) {
    const long long o = at;
    at += round256(n);
    return o;
  };
  p.starts = take(p.direct ? 0 : 2 * bg * (a.nb + 1));
  p.lists = take(p.direct ? 0 : 2 * bg * 64 * a.topk);
  p.vexp = take((long long)a.batch * a.kv * std::max(1, a.nb) * p.subs);
  p.ml = take(8 * rows * p.slots);
  const long long cq = p.direct ? a.nq : 64LL * p.chunk;
  p.part = take((long long)part_bytes * a.batch * a.heads * cq * p.slots * p.dvp);
  p.low = take(part_bytes == 2 ? 2LL * a.batch * a.heads * cq * p.slots * p.dvp : 0);
  p.all = at;
  return p;
}

static int check_attend(const BlockArgs& a, const AttendPlan& p) {
  const long long bh = (long long)a.batch * a.kv;
  bool fits;
  if (p.few) {
    fits = fits_grid(bh * a.nq * ((a.group + 15) / 16), 512);
  } else {
    const long long nrange = p.direct ? 0 : (p.chunk + p.range - 1) / p.range;
    const long long queries = p.direct ? a.nq : std::min<long long>(a.nq, 64LL * p.chunk);
    fits = fits_grid((long long)a.batch * queries * a.heads * (p.dvp / 8) + 255, 1) &&
           (p.direct ? fits_grid(bh * a.nq * a.topk * p.subs, 64) : fits_grid(bh * nrange * a.nb * p.subs, 256) && fits_grid(bh * p.groups, 64));
  }
  return fits ? 0 : fail(-3, "block_attention: more queries or blocks than one launch covers");
}

template <typename T, int KEYS, int DK32, int DV16>
static int attend_launch(const AttendArgs& p, bool direct, bool few, hipStream_t s) {
  const BlockArgs& a = p.a;
  const long long bh = (long long)a.batch * a.kv;
  if (few) {
    const int nw = std::min(8, p.slots), lds = nw * DV16 * 16 * (KEYS + 8) * 2;
    auto kern = block_attend_few_kernel<T, KEYS, DK32, DV16>;
    if (int rc = allow_big_lds(reinterpret_cast<const void*>(kern), 8 * DV16 * 16 * (KEYS + 8) * 2)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(bh * a.nq * ((a.group + 15) / 16))), dim3(64 * nw), lds, s, p);  // (no more than the rows)
    YL_HIP(hipGetLastError());
    return 0;
  }
  const long long wg = direct ? bh * a.nq * a.topk * p.subs : bh * p.nrange * a.nb * p.subs;
  if (direct)
    hipLaunchKernelGGL((block_attend_kernel<T, KEYS, DK32, DV16, true>), dim3((unsigned)wg), dim3(64), 0, s, p);
  else
    hipLaunchKernelGGL((block_attend_kernel<T, KEYS, DK32, DV16, false>), dim3((unsigned)wg), dim3(256), (size_t)256 * p.range, s, p);
  YL_HIP(hipGetLastError());
  return 0;
}
template <typename T, int KEYS>
static int attend_by_width(const AttendArgs& p, bool direct, bool few, hipStream_t s) {
  const int dk = p.a.dk;
  if (p.a.dv <= 64) {
    if (dk <= 32) return attend_launch<T, KEYS, 1, 4>(p, direct, few, s);
    return dk <= 64 ? attend_launch<T, KEYS, 2, 4>(p, direct, few, s) : attend_launch<T, KEYS, 4, 4>(p, direct, few, s);
  }
  if (dk <= 32) return attend_launch<T, KEYS, 1, 8>(p, direct, few, s);
  return dk <= 64 ? attend_launch<T, KEYS, 2, 8>(p, direct, few, s) : attend_launch<T, KEYS, 4, 8>(p, direct, few, s);
}

extern "C" int64_t yl_block_attention_workspace_bytes(int dtype, int batch, int nq, int nk, int heads, int kv_heads, int dk, int dv, int block,
                                                      int topk) {
  BlockArgs a{};
  yl_heads dummy{reinterpret_cast<void*>(16), 0, 0, 0};
  if (fill_args("block_attention", &dummy, &dummy, dtype, batch, nq, nk, heads, kv_heads, dk, block, topk, nullptr, 0, &a)) return -1;
  if (dv < 8 || dv > 128 || dv % 8) {
    fail(-3, "block_attention: value widths are multiples of 8 up to 128");
    return -1;
  }
  if (batch * (long long)nq == 0) return 0;
  const AttendPlan p = plan_attend(a, dv, dtype);
  return check_attend(a, p) ? -1 : p.all;
}

// the attention of `p.a` (sizes, tensors, picked and scale filled in), with plan `pl` and its workspace
static int attend_run(AttendArgs& p, const AttendPlan& pl, int dtype, char* w, hipStream_t s) {
  BlockArgs& a = p.a;
  const int batch = a.batch, nq = a.nq, heads = a.heads, kv_heads = a.kv, block = a.block;
  p.subs = pl.subs, p.slots = pl.slots, p.groups = pl.groups, p.range = pl.range;
  p.gn = pl.groups, p.cq = pl.direct ? nq : 64 * pl.chunk;
  p.mlrow = (long long)nq * a.group;
  p.q32 = a.q.st < (1 << 24) && a.q.sh < (1 << 24) && 4096 * a.q.st + 1024 * a.q.sh < (1LL << 31);
  p.starts = reinterpret_cast<unsigned short*>(w + pl.starts), p.lists = reinterpret_cast<unsigned short*>(w + pl.lists);
  p.vexp = reinterpret_cast<signed char*>(w + pl.vexp), p.part = w + pl.part, p.low = pl.low - pl.part, p.ml = reinterpret_cast<float2*>(w + pl.ml);
  if (!pl.direct) {
    hipLaunchKernelGGL(block_lists_kernel, dim3((unsigned)(batch * kv_heads * pl.groups)), dim3(64), (size_t)a.nb * 10 + 16, s, p);
    YL_HIP(hipGetLastError());
  }
  return by_type16(dtype, [&](auto* t) {
    typedef BA_T(t) T;
    if (pl.few) return block == 32 ? attend_by_width<T, 32>(p, true, true, s) : attend_by_width<T, 64>(p, true, true, s);
    for (int g0 = 0; g0 < pl.groups; g0 += pl.chunk) {
      p.g0 = g0, p.gn = std::min(pl.chunk, pl.groups - g0);
      p.nrange = (p.gn + pl.range - 1) / pl.range;
      if (a.nb > 0 || pl.direct)
        if (int rc = block == 32 ? attend_by_width<T, 32>(p, pl.direct, false, s) : attend_by_width<T, 64>(p, pl.direct, false, s)) return rc;
      const long long items = (long long)batch * std::min(64 * p.gn, nq - 64 * g0) * heads * (pl.dvp / 8);
      const dim3 grid((unsigned)((items + 255) / 256));
      typedef typename Vec<T>::part P;
      if (pl.direct && pl.dvp == 64) hipLaunchKernelGGL((block_join_kernel<T, float, 64>), grid, dim3(256), 0, s, p);
      else if (pl.direct) hipLaunchKernelGGL((block_join_kernel<T, float, 128>), grid, dim3(256), 0, s, p);
      else if (pl.dvp == 64) hipLaunchKernelGGL((block_join_kernel<T, P, 64>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((block_join_kernel<T, P, 128>), grid, dim3(256), 0, s, p);
      YL_HIP(hipGetLastError());
    }
    return 0;
  });
}

extern "C" int yl_block_attention(const yl_heads* q, const yl_heads* k, const yl_heads* v, int dtype, int batch, int nq, int nk,
                                  int heads, int kv_heads, int dk, int dv, int block, int topk, const int32_t* picked,
                                  const uint8_t* mask, int64_t mask_stride, float scale, const yl_heads* out, void* work,
                                  int64_t work_bytes, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  AttendArgs p{};
  BlockArgs& a = p.a;
  if (int rc = fill_args("block_attention", q, k, dtype, batch, nq, nk, heads, kv_heads, dk, block, topk, mask, mask_stride, &a)) return rc;
  if (dv < 8 || dv > 128 || dv % 8) return fail(-3, "block_attention: value widths are multiples of 8 up to 128");
  if (batch * (long long)nq == 0) return 0;
  if (nk > 0)
    if (int rc = check_heads("block_attention", "v", v)) return rc;
  if (int rc = check_heads("block_attention", "out", out)) return rc;
  if ((batch > 1 && out->batch == 0) || (nq > 1 && out->token == 0) || (heads > 1 && out->head == 0))
    return fail(-1, "block_attention: out has a stride of 0");
  if (!picked) return fail(-1, "block_attention: null pointer");
  const AttendPlan pl = plan_attend(a, dv, dtype);
  if (int rc = check_attend(a, pl)) return rc;
  if (pl.all > 0 && (!work || work_bytes < pl.all || (reinterpret_cast<uintptr_t>(work) & 15)))
    return fail(-1, "block_attention: workspace missing, too small or not 16-byte aligned");
  if (nk > 0) a.v = Heads{v->data, v->batch, v->token, v->head, 8};
  a.o = Heads{out->data, out->batch, out->token, out->head, 8};
  a.dv = dv, a.scale = scale, a.picked = const_cast<int32_t*>(picked);
  return attend_run(p, pl, dtype, static_cast<char*>(work), s);
}

// ---- YL_OP_ATTENTION on the network's maps: q (32) | k (32) | v (64) channels of every head, all tokens of an image
static BlockArgs map_args(int batch, int heads, int n, int block, int topk) {
  BlockArgs a{};
  a.batch = batch, a.nq = a.nk = n, a.heads = a.kv = heads, a.group = 1, a.magic = 1;
  a.dk = 32, a.dv = 64, a.block = block, a.nb = (n + block - 1) / block, a.topk = topk;
  fill_errors(&a);
  return a;
}
namespace yl {
long long block_attention_map_bytes(int batch, int heads, int n, int block, int topk) {
  BlockArgs a = map_args(batch, heads, n, block, topk);
  return round256(4LL * batch * heads * n * topk) + std::max(plan_select(&a).all, plan_attend(a, a.dv, YL_BF16).all);
}
int block_attention_map_launch(const AttnArgs& t, int block, int topk, char* work, hipStream_t s) {
  AttendArgs p{};
  BlockArgs& a = p.a;
  a = map_args(t.batch, t.heads, t.N, block, topk);
  a.W = t.W;
  auto heads = [&](const PView& v, int plane, int per_head) {
    return Heads{v.base + plane * v.plane + v.g0 * 8LL, v.img * 8LL, 8, per_head * v.plane, v.plane};
  };
  a.q = heads(t.in, 0, 16), a.k = heads(t.in, 4, 16), a.v = heads(t.in, 8, 16), a.o = heads(t.out, 0, 8);
  a.scale = t.scale;
  a.picked = reinterpret_cast<int*>(work);
  char* const w = work + round256(4LL * a.batch * a.kv * a.nq * a.topk);
  const SelectPlan sp = plan_select(&a);
  if (int rc = select_run(a, sp, YL_BF16, w, s)) return rc;
  return attend_run(p, plan_attend(a, a.dv, YL_BF16), YL_BF16, w, s);
}
}  // namespace yl

extern "C" int64_t yl_attention_scratch_bytes(int batch, int heads, int tokens, int block, int topk) {
  if (batch < 1 || heads < 1 || tokens < 1 || (block != 32 && block != 64 && block != 128) || topk < 1 || topk > BA_MAX_TOPK ||
      ((long long)tokens + block - 1) / block > BA_MAX_BLOCKS || !yl::fits31(batch, heads, tokens)) {
    fail(-3, "attention: blocks of 32, 64 or 128 tokens, at most 4096 of them, 1 to 64 for a token");
    return -1;
  }
  const BlockArgs a = map_args(batch, heads, tokens, block, topk);
  if (check_select(a) || check_attend(a, plan_attend(a, a.dv, YL_BF16))) return -1;
  return yl::block_attention_map_bytes(batch, heads, tokens, block, topk);
}
