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
// One wave per (image, query, head): a lane per key for the scores, a lane per value channel for the sum.
template <typename T>
__global__ __launch_bounds__(64) void block_attention_kernel(BlockArgs a) {
  __shared__ float qs[128];
  __shared__ float p[64];
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;  // (b * nq + i) * heads + head
  const int head = (int)(row % a.heads);
  const long long bi = row / a.heads;
  const int i = (int)(bi % a.nq), b = (int)(bi / a.nq), h = head / a.group;
  const float ninf = -__builtin_huge_valf();
  for (int d = lane; d < a.dk; d += 64)
    qs[d] = (float)(static_cast<const T*>(a.q.p) + b * a.q.sb + i * a.q.st + head * a.q.sh)[d] * (a.scale * 1.44269504088896340736f);
  __syncthreads();
  const int* pick = a.picked + (((long long)b * a.kv + h) * a.nq + i) * a.topk;
  float m = ninf, l = 0.f, acc[2] = {0.f, 0.f};
  for (int t = 0; t < a.topk; ++t) {
    const int j = pick[t];
    bool skip = j < 0 || j >= a.nb;
    for (int u = 0; u < t && !skip; ++u) skip = pick[u] == j;  // a block counts once
    if (skip) continue;
    for (int c0 = 0; c0 < a.block; c0 += 64) {
      const int kk = j * a.block + c0 + lane;
      const bool ok = c0 + lane < a.block && kk < a.nk && (!a.mask || a.mask[b * a.mask_stride + kk]);
      float s = ninf;
      if (ok) {
        const T* kp = static_cast<const T*>(a.k.p) + b * a.k.sb + kk * a.k.st + h * a.k.sh;
        s = 0.f;
        for (int d = 0; d < a.dk; ++d) s += qs[d] * (float)kp[d];
      }
      const unsigned long long any = __ballot(ok);
      if (!any) continue;
      float mx = s;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      const float mn = fmaxf(m, mx);
      const float base = mn == ninf ? 0.f : mn;  // (every score -inf: exponentials of -inf, all 0)
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      const float e = ok ? __builtin_amdgcn_exp2f(s - base) : 0.f;
      float sum = e;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
      l = l * alpha + sum;
      m = mn;
      __syncthreads();
      p[lane] = e;
      __syncthreads();
      acc[0] *= alpha, acc[1] *= alpha;
      for (int u = 0; u < 64; ++u) {
        if (!(any >> u & 1)) continue;
        const T* vp = static_cast<const T*>(a.v.p) + b * a.v.sb + (long long)(j * a.block + c0 + u) * a.v.st + h * a.v.sh;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (lane + 64 * x < a.dv) acc[x] += p[u] * (float)vp[lane + 64 * x];
      }
    }
  }
  T* op = static_cast<T*>(const_cast<void*>(a.o.p)) + b * a.o.sb + i * a.o.st + head * a.o.sh;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (lane + 64 * x < a.dv) op[lane + 64 * x] = (T)(l == 0.f ? 0.f : acc[x] / l);
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

extern "C" int64_t yl_block_attention_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dk, int dv, int block,
                                                      int topk) {
  BlockArgs a{};
  yl_heads dummy{reinterpret_cast<void*>(16), 0, 0, 0};
  if (fill_args("block_attention", &dummy, &dummy, YL_BF16, batch, nq, nk, heads, kv_heads, dk, block, topk, nullptr, 0, &a)) return -1;
  if (dv < 8 || dv > 128 || dv % 8) return fail(-1, "block_attention: value widths are multiples of 8 up to 128");
  return 0;
}

extern "C" int yl_block_attention(const yl_heads* q, const yl_heads* k, const yl_heads* v, int dtype, int batch, int nq, int nk,
                                  int heads, int kv_heads, int dk, int dv, int block, int topk, const int32_t* picked,
                                  const uint8_t* mask, int64_t mask_stride, float scale, const yl_heads* out, void* work,
                                  int64_t work_bytes, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  BlockArgs a{};
  if (int rc = fill_args("block_attention", q, k, dtype, batch, nq, nk, heads, kv_heads, dk, block, topk, mask, mask_stride, &a)) return rc;
  if (dv < 8 || dv > 128 || dv % 8) return fail(-3, "block_attention: value widths are multiples of 8 up to 128");
  if (batch * (long long)nq == 0) return 0;
  if (nk > 0)
    if (int rc = check_heads("block_attention", "v", v)) return rc;
  if (int rc = check_heads("block_attention", "out", out)) return rc;
  if (!picked) return fail(-1, "block_attention: null pointer");
  const long long need = yl_block_attention_workspace_bytes(batch, nq, nk, heads, kv_heads, dk, dv, block, topk);
  if (need > 0 && (!work || work_bytes < need || (reinterpret_cast<uintptr_t>(work) & 15)))
    return fail(-1, "block_attention: workspace missing, too small or not 16-byte aligned");
  if (nk > 0) a.v = Heads{v->data, v->batch, v->token, v->head};
  a.o = Heads{out->data, out->batch, out->token, out->head};
  a.dv = dv, a.scale = scale, a.picked = const_cast<int32_t*>(picked);
  return by_type16(dtype, [&](auto* t) {
    hipLaunchKernelGGL(block_attention_kernel<BA_T(t)>, dim3(batch * nq * heads), dim3(64), 0, s, a);
    YL_HIP(hipGetLastError());
    return 0;
  });
}
