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
#include <type_traits>

#include "conv_common.h"

namespace yl {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BA_MAX_BLOCKS = 4096;  // key blocks per image: the exact selection keeps a row of 64-bit keys in LDS (32 KB)
constexpr int BA_MAX_TOPK = 64;

// element (b, t, h, c) of a tensor of heads: p + b * sb + t * st + h * sh + c
struct Heads {
  const void* p;
  long long sb, st, sh;
};

struct BlockArgs {
  Heads q, k, v, o;
  int batch, nq, nk, heads, kv, group;  // group = heads / kv
  int dk, dv, block, nb, topk;
  const uint8_t* mask;  // [batch][nk], row stride mask_stride; nullptr: every key may be read
  long long mask_stride;
  float scale;
  double* mean;   // [batch][kv][dk][nb]
  int* count;     // [batch][nb]: unmasked keys of a block
  int* picked;    // [batch][kv][nq][topk]
};

// ------------------------------------------------------------------------------------------------ block means
// One workgroup per (image, kv head, block): thread = (key lane, 8 dims).
template <typename T>
__global__ __launch_bounds__(256) void block_mean_kernel(BlockArgs a) {
  __shared__ double sum[256 * 8];
  __shared__ int cnt;
  const int j = blockIdx.x % a.nb, bh = blockIdx.x / a.nb, h = bh % a.kv, b = bh / a.kv;
  const int C = a.dk >> 3, KL = 256 / C;
  const int c = threadIdx.x % C, kl = threadIdx.x / C;
  const int k0 = j * a.block, kn = min(a.block, a.nk - k0);
  if (threadIdx.x == 0) cnt = 0;
  __syncthreads();
  double acc[8] = {};
  int mine = 0;
  typedef T t8 __attribute__((ext_vector_type(8)));
  if (kl < KL)
    for (int i = kl; i < kn; i += KL) {
      if (a.mask && !a.mask[b * a.mask_stride + k0 + i]) continue;
      ++mine;
      const t8 x = *reinterpret_cast<const t8*>(static_cast<const T*>(a.k.p) + b * a.k.sb + (long long)(k0 + i) * a.k.st + h * a.k.sh + c * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += (double)(float)x[e];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (kl < KL) sum[(kl * C + c) * 8 + e] = acc[e];
  if (c == 0 && mine) atomicAdd(&cnt, mine);  // (whole numbers: the order does not matter)
  __syncthreads();
  const int n = cnt;
  for (int d = threadIdx.x; d < a.dk; d += 256) {
    double s = 0;
    for (int i = 0; i < KL; ++i) s += sum[i * a.dk + d];
    a.mean[((long long)bh * a.dk + d) * a.nb + j] = n ? s / n : 0.0;
  }
  if (h == 0 && threadIdx.x == 0) a.count[b * a.nb + j] = n;
}

// ------------------------------------------------------------------------------------------------ selection
// Scores in the order of unsigned integers; 0: the block cannot be selected.  NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ unsigned long long order_key(double s, bool can) {
  if (!can) return 0;
  if (s != s) s = -__builtin_inf();
  const unsigned long long b = (unsigned long long)__double_as_longlong(s + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// One wave per (image, kv head, query): all scores in 64 bits, the topk-th largest by its bits, then the blocks at or over it.
template <typename T>
__global__ __launch_bounds__(64) void block_select_kernel(BlockArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sel_sm[];
  double* qs = reinterpret_cast<double*>(sel_sm);                                   // [dk]
  unsigned long long* key = reinterpret_cast<unsigned long long*>(sel_sm) + a.dk;   // [nb]
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;  // (b * kv + h) * nq + i
  const int i = (int)(row % a.nq);
  const int bh = (int)(row / a.nq), h = bh % a.kv, b = bh / a.kv;
  for (int d = lane; d < a.dk; d += 64) {
    double s = 0;
    for (int g = 0; g < a.group; ++g)
      s += (double)(float)(static_cast<const T*>(a.q.p) + b * a.q.sb + i * a.q.st + (long long)(h * a.group + g) * a.q.sh)[d];
    qs[d] = s;
  }
  __syncthreads();
  int can = 0;
  for (int j = lane; j < a.nb; j += 64) {
    double s = 0;
    const double* m = a.mean + (long long)bh * a.dk * a.nb + j;
    for (int d = 0; d < a.dk; ++d) s += qs[d] * m[(long long)d * a.nb];
    const bool ok = a.count[b * a.nb + j] > 0;
    can += ok;
    key[j] = order_key(s, ok);
  }
  __syncthreads();
  auto total = [&](int c) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o);
    return c;
  };
  const int n = min(a.topk, total(can));
  unsigned long long v = 0;
  int over = 0;  // keys > v that are taken whatever their index
  if (n > 0) {
    bool exact = false;
    for (int bit = 63; bit >= 0 && !exact; --bit) {
      const unsigned long long t = v | 1ull << bit;
      int c = 0;
      for (int j = lane; j < a.nb; j += 64) c += key[j] >= t;
      c = total(c);
      if (c >= n) v = t;
      exact = c == n;
    }
    int c = 0;
    for (int j = lane; j < a.nb; j += 64) c += key[j] > v;
    over = total(c);
  }
  int* out = a.picked + row * a.topk;
  int at = 0, ties = n - over;  // of the keys equal to v the first `ties` belong to the set
  for (int j0 = 0; j0 < a.nb && n > 0; j0 += 64) {
    const int j = j0 + lane;
    const unsigned long long k = j < a.nb ? key[j] : 0;
    const unsigned long long below = (1ull << lane) - 1;
    const unsigned long long eq = __ballot(j < a.nb && k == v);
    const bool take = (j < a.nb && k > v) || (j < a.nb && k == v && __popcll(eq & below) < ties);
    ties -= min(ties, (int)__popcll(eq));
    const unsigned long long all = __ballot(take);
    if (take) out[at + __popcll(all & below)] = j;
    at += __popcll(all);
  }
  for (int t = n + lane; t < a.topk; t += 64) out[t] = -1;
}

// ------------------------------------------------------------------------------------------------ attention
// Queries that pick their blocks one by one share no tile of keys.  Turned round they do: a workgroup takes ONE block (its keys in
// the registers of every wave, its values through LDS) and gathers the queries that picked it, 16 (query, head) rows to an MFMA
// tile -- S^T = K Q^T, softmax over the block, O^T = V^T P^T, where the S^T accumulators of two 16-key tiles are, after exp2, the B
// fragment of the second product -- and writes the block's normalised result of each row with its maximum and sum; a second launch
// joins a row's blocks.  Keys are read once per block and range of queries instead of once per query; the price is that every (row,
// block) result passes through memory, which is what bounds the stage (2 (dv + 4) bytes written and read per row and block).
//
// Results of a block are rounded to the tensors' type between the launches: as exact as the weights P themselves, which the matrix
// pipe takes in that type, and half the traffic; maxima, sums and the joining are fp32.
//
// Lists: 64 queries form a group; lists[group] holds its (query, slot) pairs sorted by block, starts[group][j] where block j's begin.
// A block of 128 keys is two units of 64 (two results per slot): one unit's fragments fill the registers.

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  typedef bf16x8 t8;
  typedef bf16x4 t4;
  static __device__ __forceinline__ f32x4 mfma(t8 a, t8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Vec<_Float16> {
  typedef f16x8 t8;
  typedef _Float16 t4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4 mfma(t8 a, t8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// the four lanes that share lane & 15: maximum, sum
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

struct AttendArgs {
  BlockArgs a;
  int subs, slots;          // units per block, results per row: topk * subs
  int groups, range, nrange;  // groups of 64 queries per image; groups of a workgroup's range; ranges
  unsigned short* starts;   // [batch * kv][groups][nb + 1]
  unsigned short* lists;    // [batch * kv][groups][64 * topk]: query (6 bits) << 6 | slot
  void* part;               // [row][slots][DVP], row = ((b * kv + h) * nq + i) * group + head in the group
  float2* ml;               // [row][slots]: maximum (log2), sum
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
  unsigned long long first = 0;  // this query's slots that count
  if (i < p.a.nq)
    for (int t = 0; t < topk; ++t) {
      const int j = pick[t];
      if (j >= 0 && j < nb && !(word[j] >> lane & 1)) {  // (only this lane sets this bit)
        atomicOr(&word[j], 1ull << lane);
        first |= 1ull << t;
      } else {
        for (int g = 0; g < p.a.group * p.subs; ++g)
          p.ml[(q * p.a.group + g / p.subs) * p.slots + t * p.subs + g % p.subs] = float2{-__builtin_huge_valf(), 0.f};
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
  if (i < p.a.nq)
    for (int t = 0; t < topk; ++t) {
      if (!(first >> t & 1)) continue;
      const int j = pick[t];
      list[start[j] + __popcll(word[j] & ((1ull << lane) - 1))] = (unsigned short)(lane << 6 | t);
    }
  for (int j = lane; j <= nb; j += 64) p.starts[at * (nb + 1) + j] = start[j];
}

// DIRECT: one wave per (image, kv head, query, slot, unit) straight from `picked` -- few queries, where lists would hold one entry.
template <typename T, int KEYS, int DK32, int DV16, bool DIRECT>
__global__ __launch_bounds__(DIRECT ? 64 : 256, 2) void block_attend_kernel(AttendArgs p) {
  typedef typename Vec<T>::t8 t8;
  typedef typename Vec<T>::t4 t4;
  constexpr int NT = DIRECT ? 64 : 256;
  constexpr int KT = KEYS / 16, KS = KEYS / 32, DVP = DV16 * 16, VP = KEYS + 8;
  __shared__ __attribute__((aligned(16))) T sVt[DVP * VP];
  __shared__ unsigned rows[DIRECT ? 1 : 4096];
  __shared__ int total;
  const BlockArgs& a = p.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, n = lane & 15;
  const float ninf = -__builtin_huge_valf();
  // ---- which block, which queries
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
      const long long row = ((long long)bh * a.nq + qdirect) * a.group;
      for (int e = lane; e < a.group; e += 64) p.ml[(row + e) * p.slots + tdirect * p.subs + sub] = float2{ninf, 0.f};
      if (p.slots == 1) {  // (nothing is joined: the result itself is zeros)
        const int b0 = bh / a.kv, h0 = bh % a.kv;
        for (int e = lane; e < a.group * a.dv; e += 64)
          (static_cast<T*>(const_cast<void*>(a.o.p)) + b0 * a.o.sb + qdirect * a.o.st + (long long)(h0 * a.group + e / a.dv) * a.o.sh)[e % a.dv] = (T)0.f;
      }
      return;
    }
    nrows = a.group;
  } else {
    j = unit % a.nb;
    unit /= a.nb;
    grp0 = unit % p.nrange * p.range;
    bh = unit / p.nrange;
    const int ng = min(p.range, p.groups - grp0);
    if (wave == 0) {  // a lane per group: its share of the list, copied behind the ones before it
      int from = 0, cnt = 0;
      const long long at = (long long)bh * p.groups + grp0 + lane;
      if (lane < ng) {
        from = p.starts[at * (a.nb + 1) + j];
        cnt = p.starts[at * (a.nb + 1) + j + 1] - from;
      }
      int x = cnt;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
      }
      if (lane == 63) total = x;
      for (int e = 0; e < cnt; ++e) rows[x - cnt + e] = (unsigned)lane << 12 | p.lists[at * (64 * a.topk) + from + e];
    }
    __syncthreads();
    nrows = total * a.group;
    if (nrows == 0) return;
  }
  const int h = bh % a.kv, b = bh / a.kv;
  const int k0 = j * a.block + sub * KEYS;
  const int kn = min(min(KEYS, a.block - sub * KEYS), a.nk - k0);  // keys of this unit; <= 0: none
  const bool lok = lane < kn && (!a.mask || a.mask[b * a.mask_stride + k0 + lane]);
  const unsigned long long ok = __ballot(lok);  // the keys that may be read
  // ---- values, transposed, keys in a row; a masked value counts as 0 whatever it holds
  const T* vb = static_cast<const T*>(a.v.p) + b * a.v.sb + h * a.v.sh;
  for (int it = tid; it < KEYS / 8 * (DVP / 8); it += NT) {
    const int c8 = it % (DVP / 8), kg = it / (DVP / 8);
    t8 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      v[u] = t8{};
      if (c8 * 8 < a.dv && (ok >> (kg * 8 + u) & 1)) v[u] = *reinterpret_cast<const t8*>(vb + (long long)(k0 + kg * 8 + u) * a.v.st + c8 * 8);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<t8*>(sVt + (c8 * 8 + e) * VP + kg * 8) = t8{v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
  }
  // ---- keys: fragments of the first product (row = key, 8 dims of group g)
  t8 kf[KT][DK32];
  const T* kb = static_cast<const T*>(a.k.p) + b * a.k.sb + h * a.k.sh;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int c = 0; c < DK32; ++c) {
      kf[t][c] = t8{};
      if (t * 16 + n < kn && (c * 4 + g) * 8 < a.dk) kf[t][c] = *reinterpret_cast<const t8*>(kb + (long long)(k0 + t * 16 + n) * a.k.st + (c * 4 + g) * 8);
    }
  unsigned okt = 0;  // this lane's keys t * 16 + 4 g + r, four bits per tile
#pragma unroll
  for (int t = 0; t < KT; ++t) okt |= (unsigned)(ok >> (t * 16 + 4 * g) & 15) << (4 * t);
  __syncthreads();
  // values: row i of tile d is channel (i / 4) (DVP / 4) + 4 d + i % 4, so that a lane ends up with DVP / 4 neighbouring channels
  t8 vf[DV16][KS];
#pragma unroll
  for (int d = 0; d < DV16; ++d)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const T* vr = sVt + ((n >> 2) * (DVP / 4) + d * 4 + (n & 3)) * VP + s * 32 + 4 * g;
      const t4 lo = *reinterpret_cast<const t4*>(vr), hi = *reinterpret_cast<const t4*>(vr + 16);
      vf[d][s] = t8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  const float scale = a.scale * 1.44269504088896340736f;
  const bool alone = DIRECT && p.slots == 1;  // a row has this one result: it is the output

  // a tile's queries: lane column n is (query, head) row f
  struct Row {
    long long q;  // query of the image
    int head, slot;
    bool live;
    t8 f[DK32];
  };
  auto fetch = [&](int tile, Row& w) __attribute__((always_inline)) {
    const int f = tile * 16 + n;
    w.live = f < nrows;
    const int fc = w.live ? f : 0;
    int e = fc;
    w.head = 0;
    if (a.group > 1) {
      e = fc / a.group;
      w.head = fc - e * a.group;
    }
    if constexpr (DIRECT) {
      w.q = qdirect;
      w.slot = tdirect;
    } else {
      const unsigned x = rows[e];
      w.q = (long long)(grp0 + (int)(x >> 12)) * 64 + (x >> 6 & 63);
      w.slot = (int)(x & 63);
    }
    const T* qp = static_cast<const T*>(a.q.p) + b * a.q.sb + w.q * a.q.st + (long long)(h * a.group + w.head) * a.q.sh;
#pragma unroll
    for (int c = 0; c < DK32; ++c) {
      w.f[c] = t8{};
      if ((c * 4 + g) * 8 < a.dk) w.f[c] = *reinterpret_cast<const t8*>(qp + (c * 4 + g) * 8);
    }
  };
  const int ntiles = (nrows + 15) >> 4;
  constexpr int NW = NT / 64;
  Row next;
  if (wave < ntiles) fetch(wave, next);
  for (int tile = wave; tile < ntiles; tile += NW) {
    const Row w = next;
    if (tile + NW < ntiles) fetch(tile + NW, next);
    f32x4 s[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DK32; ++c) s[t] = Vec<T>::mfma(kf[t][c], w.f[c], s[t]);
    }
    float m = ninf;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] = okt >> (4 * t + r) & 1 ? s[t][r] * scale : ninf;
        m = fmaxf(m, s[t][r]);
      }
    m = quad_max(m);
    const float base = m == ninf ? 0.f : m;  // (no key, or every score -inf: all weights 0)
    float l = 0.f;
    t8 pf[KS];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[t][r] - base);
        l += e;
        pf[t >> 1][(t & 1) * 4 + r] = (T)e;
      }
    l = quad_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    f32x4 o[DV16];
#pragma unroll
    for (int d = 0; d < DV16; ++d) {
      o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) o[d] = Vec<T>::mfma(vf[d][x], pf[x], o[d]);
    }
    if (!w.live) continue;
    const long long row = (((long long)bh) * a.nq + w.q) * a.group + w.head;
    const int slot = w.slot * p.subs + sub;
    T* dst = alone ? static_cast<T*>(const_cast<void*>(a.o.p)) + b * a.o.sb + w.q * a.o.st + (long long)(h * a.group + w.head) * a.o.sh
                   : static_cast<T*>(p.part) + (row * p.slots + slot) * DVP;
#pragma unroll
    for (int d = 0; d < DV16; d += 2) {
      const int c = g * (DVP / 4) + d * 4;
      const t8 y = {(T)(o[d][0] * inv), (T)(o[d][1] * inv), (T)(o[d][2] * inv), (T)(o[d][3] * inv),
                    (T)(o[d + 1][0] * inv), (T)(o[d + 1][1] * inv), (T)(o[d + 1][2] * inv), (T)(o[d + 1][3] * inv)};
      if (!alone || c < a.dv) *reinterpret_cast<t8*>(dst + c) = y;
    }
    if (!alone && g == 0) p.ml[row * p.slots + slot] = float2{m, l};
  }
}

// out = the slots' results weighted by their sums; one thread per (row, 8 channels)
template <typename T, int DVP>
__global__ __launch_bounds__(256) void block_join_kernel(AttendArgs p) {
  typedef typename Vec<T>::t8 t8;
  const BlockArgs& a = p.a;
  constexpr int C = DVP / 8;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(item % C) * 8;
  const long long row = item / C;
  if (row >= (long long)a.batch * a.nq * a.heads || c >= a.dv) return;
  const float2* ml = p.ml + row * p.slots;
  float m = -__builtin_huge_valf();
  for (int t = 0; t < p.slots; ++t) m = fmaxf(m, ml[t].x);
  const float base = m == -__builtin_huge_valf() ? 0.f : m;
  float acc[8] = {}, sum = 0.f;
  for (int t = 0; t < p.slots; ++t) {
    const float w = ml[t].y * __builtin_amdgcn_exp2f(ml[t].x - base);
    if (w == 0.f) continue;  // (nothing was stored for a slot without a block)
    sum += w;
    const t8 y = *reinterpret_cast<const t8*>(static_cast<const T*>(p.part) + (row * p.slots + t) * DVP + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += w * (float)y[e];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int gh = (int)(row % a.group);
  const long long q = row / a.group;
  const int i = (int)(q % a.nq), bh = (int)(q / a.nq);
  t8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (T)(acc[e] * inv);
  *reinterpret_cast<t8*>(static_cast<T*>(const_cast<void*>(a.o.p)) + bh / a.kv * a.o.sb + i * a.o.st +
                         (long long)(bh % a.kv * a.group + gh) * a.o.sh + c) = y;
}

// ------------------------------------------------------------------------------------------------ host
static long long round256(long long n) { return (n + 255) / 256 * 256; }

static int check_heads(const std::string& who, const char* name, const yl_heads* t) {
  if (!t || !t->data) return fail(-1, who + ": null " + name);
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) || ((t->batch | t->token | t->head) & 7))
    return fail(-1, who + ": " + name + " must be 16-byte aligned with strides that are multiples of 8 elements");
  if (t->batch < 0 || t->token < 0 || t->head < 0) return fail(-1, who + ": " + name + " has a negative stride");
  return 0;
}

// sizes that the calls share -> BlockArgs; nothing is launched where batch * nq is 0
static int fill_args(const std::string& who, const yl_heads* q, const yl_heads* k, int dtype, int batch, int nq, int nk, int heads,
                     int kv_heads, int dk, int block, int topk, const uint8_t* mask, int64_t mask_stride, BlockArgs* a) {
  if (dtype != YL_BF16 && dtype != YL_F16) return fail(-1, who + ": bf16 or fp16 tensors");
  if (batch < 0 || nq < 0 || nk < 0) return fail(-1, who + ": a negative size");
  if (heads < 1 || kv_heads < 1 || heads % kv_heads) return fail(-1, who + ": the query heads must be a multiple of the kv heads");
  if (dk < 8 || dk > 128 || dk % 8) return fail(-3, who + ": key widths are multiples of 8 up to 128");
  if (block != 32 && block != 64 && block != 128) return fail(-3, who + ": blocks of 32, 64 or 128 keys");
  if (topk < 1 || topk > BA_MAX_TOPK) return fail(-3, who + ": 1 to 64 blocks for a query");
  const long long nb = ((long long)nk + block - 1) / block;
  if (nb > BA_MAX_BLOCKS) return fail(-3, who + ": more than 4096 key blocks");
  if ((long long)batch * heads * nq > 0x7FFFFFFFLL || (long long)batch * kv_heads * nb > 0x7FFFFFFFLL)
    return fail(-3, who + ": more rows or blocks than one launch covers");
  if (batch * (long long)nq == 0) return 0;
  if (int rc = check_heads(who, "q", q)) return rc;
  if (nk > 0)
    if (int rc = check_heads(who, "k", k)) return rc;
  if (mask && batch > 1 && mask_stride < nk) return fail(-1, who + ": the mask's row stride is smaller than a row");
  a->q = Heads{q->data, q->batch, q->token, q->head};
  if (nk > 0) a->k = Heads{k->data, k->batch, k->token, k->head};
  a->batch = batch, a->nq = nq, a->nk = nk, a->heads = heads, a->kv = kv_heads, a->group = heads / kv_heads;
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

extern "C" int64_t yl_block_select_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dk, int block) {
  BlockArgs a{};
  yl_heads dummy{reinterpret_cast<void*>(16), 0, 0, 0};
  if (fill_args("block_select", &dummy, &dummy, YL_BF16, batch, nq, nk, heads, kv_heads, dk, block, 1, nullptr, 0, &a)) return -1;
  return round256(8LL * batch * kv_heads * dk * a.nb) + round256(4LL * batch * a.nb);
}

extern "C" int yl_block_select(const yl_heads* q, const yl_heads* k, int dtype, int batch, int nq, int nk, int heads, int kv_heads,
                               int dk, int block, int topk, const uint8_t* mask, int64_t mask_stride, int32_t* picked, void* work,
                               int64_t work_bytes, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  BlockArgs a{};
  if (int rc = fill_args("block_select", q, k, dtype, batch, nq, nk, heads, kv_heads, dk, block, topk, mask, mask_stride, &a)) return rc;
  if (batch * (long long)nq == 0) return 0;
  if (!picked) return fail(-1, "block_select: null pointer");
  const long long need = yl_block_select_workspace_bytes(batch, nq, nk, heads, kv_heads, dk, block);
  if (need > 0 && (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15)))
    return fail(-1, "block_select: workspace missing, too small or not 16-byte aligned");
  a.picked = picked;
  a.mean = static_cast<double*>(work);
  a.count = reinterpret_cast<int*>(static_cast<char*>(work) + round256(8LL * batch * kv_heads * dk * a.nb));
  return by_type16(dtype, [&](auto* t) {
    if (a.nb > 0) {
      hipLaunchKernelGGL(block_mean_kernel<BA_T(t)>, dim3(batch * kv_heads * a.nb), dim3(256), 0, s, a);
      YL_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(block_select_kernel<BA_T(t)>, dim3(batch * kv_heads * nq), dim3(64), (size_t)(a.dk + a.nb) * 8, s, a);
    YL_HIP(hipGetLastError());
    return 0;
  });
}

// ---- how the attention runs: sizes, and where things lie in the workspace
struct AttendPlan {
  bool direct;
  int subs, slots, groups, range, nrange, dvp;
  long long starts, lists, part, ml, all;  // byte offsets
};

static AttendPlan plan_attend(const BlockArgs& a, int dv) {
  AttendPlan p{};
  p.subs = a.block == 128 ? 2 : 1;
  p.slots = a.topk * p.subs;
  p.dvp = dv <= 64 ? 64 : 128;
  p.groups = (a.nq + 63) / 64;
  // the lists pay where a block is picked often; below that, a wave per (query, block)
  p.direct = a.nq <= 4 || (long long)a.nq * a.topk <= 2LL * a.nb;
  // a workgroup's range of queries: about 256 (query, head) rows, 16 tiles, for an average block
  const long long per64 = 64LL * a.topk * a.group;
  p.range = (int)std::min<long long>(64, std::max<long long>(1, 256LL * std::max(1, a.nb) / per64));
  p.range = std::min(p.range, p.groups);
  p.nrange = p.range ? (p.groups + p.range - 1) / p.range : 0;
  const long long rows = (long long)a.batch * a.nq * a.heads, bg = (long long)a.batch * a.kv * p.groups;
  long long at = 0;
  auto take = [&](long long n) {
    const long long o = at;
    at += round256(n);
    return o;
  };
  p.starts = take(p.direct ? 0 : 2 * bg * (a.nb + 1));
  p.lists = take(p.direct ? 0 : 2 * bg * 64 * a.topk);
  p.ml = take(8 * rows * p.slots);
  p.part = take(p.slots == 1 && p.direct ? 0 : 2 * rows * p.slots * p.dvp);
  p.all = at;
  return p;
}

template <typename T, int KEYS, int DK32, int DV16>
static int attend_launch(const AttendArgs& p, bool direct, hipStream_t s) {
  const BlockArgs& a = p.a;
  const long long bh = (long long)a.batch * a.kv;
  const long long wg = direct ? bh * a.nq * a.topk * p.subs : bh * p.nrange * a.nb * p.subs;
  if (wg > 0x7FFFFFFFLL) return fail(-3, "block_attention: more blocks and queries than one launch covers");
  if (direct)
    hipLaunchKernelGGL((block_attend_kernel<T, KEYS, DK32, DV16, true>), dim3((unsigned)wg), dim3(64), 0, s, p);
  else
    hipLaunchKernelGGL((block_attend_kernel<T, KEYS, DK32, DV16, false>), dim3((unsigned)wg), dim3(256), 0, s, p);
  YL_HIP(hipGetLastError());
  return 0;
}
template <typename T, int KEYS>
static int attend_by_width(const AttendArgs& p, bool direct, hipStream_t s) {
  const int dk = p.a.dk;
  if (p.a.dv <= 64)
    return dk <= 32 ? attend_launch<T, KEYS, 1, 4>(p, direct, s) : dk <= 64 ? attend_launch<T, KEYS, 2, 4>(p, direct, s) : attend_launch<T, KEYS, 4, 4>(p, direct, s);
  return dk <= 32 ? attend_launch<T, KEYS, 1, 8>(p, direct, s) : dk <= 64 ? attend_launch<T, KEYS, 2, 8>(p, direct, s) : attend_launch<T, KEYS, 4, 8>(p, direct, s);
}

extern "C" int64_t yl_block_attention_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dk, int dv, int block,
                                                      int topk) {
  BlockArgs a{};
  yl_heads dummy{reinterpret_cast<void*>(16), 0, 0, 0};
  if (fill_args("block_attention", &dummy, &dummy, YL_BF16, batch, nq, nk, heads, kv_heads, dk, block, topk, nullptr, 0, &a)) return -1;
  if (dv < 8 || dv > 128 || dv % 8) {
    fail(-3, "block_attention: value widths are multiples of 8 up to 128");
    return -1;
  }
  return batch * (long long)nq == 0 ? 0 : plan_attend(a, dv).all;
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
  if (!picked) return fail(-1, "block_attention: null pointer");
  const AttendPlan pl = plan_attend(a, dv);
  if (!work || work_bytes < pl.all || (reinterpret_cast<uintptr_t>(work) & 15))
    return fail(-1, "block_attention: workspace missing, too small or not 16-byte aligned");
  if (nk > 0) a.v = Heads{v->data, v->batch, v->token, v->head};
  a.o = Heads{out->data, out->batch, out->token, out->head};
  a.dv = dv, a.scale = scale, a.picked = const_cast<int32_t*>(picked);
  char* const w = static_cast<char*>(work);
  p.subs = pl.subs, p.slots = pl.slots, p.groups = pl.groups, p.range = pl.range, p.nrange = pl.nrange;
  p.starts = reinterpret_cast<unsigned short*>(w + pl.starts), p.lists = reinterpret_cast<unsigned short*>(w + pl.lists);
  p.part = w + pl.part, p.ml = reinterpret_cast<float2*>(w + pl.ml);
  if (!pl.direct) {
    hipLaunchKernelGGL(block_lists_kernel, dim3((unsigned)(batch * kv_heads * pl.groups)), dim3(64), (size_t)a.nb * 10 + 16, s, p);
    YL_HIP(hipGetLastError());
  }
  return by_type16(dtype, [&](auto* t) {
    typedef BA_T(t) T;
    if (a.nb > 0 || pl.direct)
      if (int rc = block == 32 ? attend_by_width<T, 32>(p, pl.direct, s) : attend_by_width<T, 64>(p, pl.direct, s)) return rc;
    if (pl.slots == 1 && pl.direct) return 0;
    const long long items = (long long)batch * nq * heads * (pl.dvp / 8);
    if (pl.dvp == 64)
      hipLaunchKernelGGL((block_join_kernel<T, 64>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((block_join_kernel<T, 128>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, p);
    YL_HIP(hipGetLastError());
    return 0;
  });
}
