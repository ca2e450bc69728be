// sample.cu -- the next token of each row of logits, from one uniform number a row.
//
// With m = max x and T the temperature, a token's weight is w = exp((x - m) / T) and its mass the whole
// number rint(w 2^40).  All sums are sums of masses: they have no order, so the token depends on the
// row, its settings and its number alone, not on how the row was split.  Tokens are ordered by logit,
// equal ones by index; every filter keeps a beginning of that order (at least its first token):
//   top-k   the first k tokens, of total mass Z_k;
//   top-p   those with less than p Z_k mass before them;
//   min-p   those with w >= min_p.
// The token is the first in vocabulary order whose inclusive mass, over the kept tokens, exceeds u Z.
//
// A filter's cut is the element of the order where the inclusive count reaches k (or the inclusive mass
// p Z_k).  It is found by digits: a histogram over 2048 bins of the distance from the maximum, then over
// the bits of the logit and of the index within the bin that holds the cut, until few enough elements
// are left to rank them directly.
#include <algorithm>
#include <cmath>

#include "attn_common.cuh"
#include "host_util.h"
#include "kata_b200.h"

namespace kata {
namespace {

constexpr int kST = 1024;    // threads per row
constexpr int kBins = 2048;
constexpr int kList = 512;   // elements ranked directly
typedef unsigned long long u64;

struct SampleParams {
  const void* logits;
  long long ld;
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  int top_k_s;
  long long* token;
  float* logprob;
  int V;
};

// Ascending in the order of tokens: the bits of -x as an unsigned number (-0 counts as 0).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
}

struct Row {
  float m, inv;  // maximum, 1 / temperature
  __device__ __forceinline__ float z(float x) const { return x == m ? 0.f : __fmul_rn(__fsub_rn(x, m), inv); }
  // a mask weighs nothing even at an infinite temperature, nor does anything beside an infinite logit
  __device__ __forceinline__ float w(float x) const {
    return x == m ? 1.f : (x == -INFINITY || m == INFINITY) ? 0.f : expf(z(x));
  }
  __device__ __forceinline__ int bin(float x) const {
    return x == m ? 0 : static_cast<int>(fminf(__fmul_rn(__fsub_rn(m, x), 64.f), static_cast<float>(kBins - 1)));
  }
};
__device__ __forceinline__ u64 mass_of(float w) { return static_cast<u64>(__float2ll_rn(w * 1099511627776.f)); }

template <typename T>
__device__ __forceinline__ float load_logit(const T* p, int i) {
  const float x = to_f32<T>(p[i]);
  return x != x ? -INFINITY : x;
}

struct Smem {
  u64 mass[kBins];
  uint32_t cnt[kBins];
  u64 lmass[kList];
  uint32_t lkey[kList], lidx[kList];
  u64 wsum[kST / 32];
  float wmax[kST / 32];
  int n_list, bin, found;
  uint32_t cut_key, cut_idx;
  u64 before;
};

__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// Finds the first token of the order whose inclusive count (BY_MASS: inclusive mass) is at least
// `limit`, which the row's total reaches.  Leaves it in s.cut_key / s.cut_idx.
template <typename T, bool BY_MASS>
__device__ void find_cut(Smem& s, const T* x, const SampleParams& p, const Row& row, u64 limit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int b1 = -1;
  uint32_t key = 0, kmask = 0, idx = 0, imask = 0;
  u64 rem = limit;
  for (int level = 0; level < 7; ++level) {
    // digits in turn: distance bin, key bits 31..21, 20..10, 9..0, index bits 31..22, 21..11, 10..0
    const int shift = level == 1 ? 21 : level == 2 ? 10 : level == 3 ? 0 : level == 4 ? 22 : level == 5 ? 11 : 0;
    const uint32_t width = (level == 3 || level == 4) ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kST) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    for (int i = tid; i < p.V; i += kST) {
      const float v = load_logit(x, i);
      const int b = row.bin(v);
      const uint32_t k = order_key(v);
      if (level > 0 && (b != b1 || ((k ^ key) & kmask) || ((static_cast<uint32_t>(i) ^ idx) & imask))) continue;
      const uint32_t d = level == 0 ? b : level <= 3 ? (k >> shift) & width : (static_cast<uint32_t>(i) >> shift) & width;
      atomicAdd(&s.cnt[d], 1u);
      if (BY_MASS) atomicAdd(&s.mass[d], mass_of(row.w(v)));
    }
    __syncthreads();
    {
      const u64 a = BY_MASS ? s.mass[2 * tid] : s.cnt[2 * tid], b = BY_MASS ? s.mass[2 * tid + 1] : s.cnt[2 * tid + 1];
      const u64 inc = warp_scan(a + b, lane);
      if (lane == 31) s.wsum[warp] = inc;
      __syncthreads();
      u64 base = 0;
      for (int w = 0; w < warp; ++w) base += s.wsum[w];
      const u64 before = base + inc - a - b;
      if (before < rem && before + a >= rem) {
        s.bin = 2 * tid;
        s.before = before;
      } else if (before + a < rem && before + a + b >= rem) {
        s.bin = 2 * tid + 1;
        s.before = before + a;
      }
      __syncthreads();
    }
    const uint32_t d = s.bin;
    rem -= s.before;
    if (level == 0) {
      b1 = d;
    } else if (level <= 3) {
      key |= d << shift;
      kmask |= width << shift;
    } else {
      idx |= d << shift;
      imask |= width << shift;
    }
    const uint32_t n = s.cnt[d];
    __syncthreads();
    if (n > kList) continue;
    // few enough: rank them
    for (int i = tid; i < p.V; i += kST) {
      const float v = load_logit(x, i);
      const uint32_t k = order_key(v);
      if (row.bin(v) != b1 || ((k ^ key) & kmask) || ((static_cast<uint32_t>(i) ^ idx) & imask)) continue;
      const int at = atomicAdd(&s.n_list, 1);
      s.lkey[at] = k;
      s.lidx[at] = i;
      s.lmass[at] = BY_MASS ? mass_of(row.w(v)) : 1ull;
    }
    __syncthreads();
    if (tid < static_cast<int>(n)) {
      u64 before = 0;
      const uint32_t k = s.lkey[tid], ix = s.lidx[tid];
      for (uint32_t j = 0; j < n; ++j)
        if (s.lkey[j] < k || (s.lkey[j] == k && s.lidx[j] < ix)) before += s.lmass[j];
      if (before < rem && before + s.lmass[tid] >= rem) {
        s.cut_key = k;
        s.cut_idx = ix;
      }
    }
    __syncthreads();
    return;
  }
}

// total * n24 / 2^24, rounded down or up
__device__ __forceinline__ u64 share(u64 total, u64 n24, bool up) {
  const u64 hi = __umul64hi(total, n24), lo = total * n24;
  return (hi << 40) + (lo >> 24) + ((up && (lo & 0xffffffull)) ? 1 : 0);
}

template <typename T>
__global__ void __launch_bounds__(kST) sample_kernel(const SampleParams p) {
  __shared__ Smem s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long b = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + b * p.ld;
  const float temp = p.temperature ? p.temperature[b] : p.temperature_s;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_s;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_s;
  int k = p.top_k ? p.top_k[b] : p.top_k_s;
  const u64 p24 = top_p > 0.f ? static_cast<u64>(fminf(top_p, 1.f) * 16777216.f) : 0;
  if (k <= 0 || k > p.V) k = p.V;
  if (!(temp > 0.f) || min_p > 1.f || p24 == 0) k = 1;  // only the first token is kept

  float m = -INFINITY;
  for (int i = tid; i < p.V; i += kST) m = fmaxf(m, load_logit(x, i));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s.wmax[warp] = m;
  __syncthreads();
  m = s.wmax[0];
  for (int w = 1; w < kST / 32; ++w) m = fmaxf(m, s.wmax[w]);
  if (m == -INFINITY) {  // nothing to draw from
    if (tid == 0) {
      p.token[b] = -1;
      p.logprob[b] = -INFINITY;
    }
    return;
  }
  const Row row{m, temp > 0.f ? 1.f / temp : 1.f};

  uint32_t cut_key = 0xffffffffu, cut_idx = 0xffffffffu;
  if (k < p.V) {
    find_cut<T, false>(s, x, p, row, k);
    cut_key = s.cut_key;
    cut_idx = s.cut_idx;
    __syncthreads();
  }
  // Mass of the kept tokens in vocabulary order; warps take consecutive ranges
  const int per = (p.V + kST / 32 - 1) / (kST / 32);
  const int lo = min(p.V, warp * per), hi = min(p.V, lo + per);
  auto kept_mass = [&](int i, bool floor) -> u64 {
    const float v = load_logit(x, i);
    const uint32_t key = order_key(v);
    if (key > cut_key || (key == cut_key && static_cast<uint32_t>(i) > cut_idx)) return 0;
    const float w = row.w(v);
    return floor && w < min_p ? 0 : mass_of(w);
  };
  auto total_mass = [&](bool floor) -> u64 {
    u64 t = 0;
    for (int i = lo + lane; i < hi; i += 32) t += kept_mass(i, floor);
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) s.wsum[warp] = t;
    __syncthreads();
    u64 all = 0;
    for (int w = 0; w < kST / 32; ++w) all += s.wsum[w];
    return all;
  };
  if (k > 1 && top_p < 1.f) {
    const u64 limit = share(total_mass(false), p24, true);
    __syncthreads();
    find_cut<T, true>(s, x, p, row, limit);
    cut_key = s.cut_key;
    cut_idx = s.cut_idx;
    __syncthreads();
  }
  const bool floor = k > 1;
  const u64 total = total_mass(floor);
  const float uu = p.u[b];
  u64 u24 = uu > 0.f ? static_cast<u64>(fminf(uu, 1.f) * 16777216.f) : 0;
  if (u24 > 16777215ull) u24 = 16777215ull;
  const u64 target = share(total, u24, false);
  u64 base = 0;
  for (int w = 0; w < warp; ++w) base += s.wsum[w];
  if (base <= target && target < base + s.wsum[warp]) {
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      const u64 inc = warp_scan(i < hi ? kept_mass(i, floor) : 0, lane) + base;
      const unsigned hit = __ballot_sync(0xffffffffu, inc > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          p.token[b] = i;
          const double z = temp > 0.f ? row.z(load_logit(x, i)) : 0.f;
          p.logprob[b] = static_cast<float>(z) - static_cast<float>(log(static_cast<double>(total) * 0x1p-40));
        }
        break;
      }
      base = __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

}  // namespace
}  // namespace kata

using namespace kata;

extern "C" int kata_sample(const kata_sample_args* a, kata_stream_t stream) {
  if (!a) return KATA_ERR_INVALID;
  if (a->dtype != KATA_DTYPE_F32 && a->dtype != KATA_DTYPE_BF16 && a->dtype != KATA_DTYPE_F16) return KATA_ERR_DTYPE;
  if (a->B < 0 || a->V < 1 || a->B > 0x7fffffff || a->V > (1 << 22)) return KATA_ERR_SHAPE;
  if (a->B > 1 && a->ld < a->V) return KATA_ERR_SHAPE;
  if (a->B == 0) return KATA_OK;
  if (!a->logits || !a->u || !a->token || !a->logprob) return KATA_ERR_INVALID;
  const size_t es = a->dtype == KATA_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->logits) % es) return KATA_ERR_ALIGN;
  SampleParams p;
  p.logits = a->logits;
  p.ld = a->ld;
  p.u = a->u;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.temperature_s = a->temperature_all;
  p.top_k_s = a->top_k_all;
  p.top_p_s = a->top_p_all;
  p.min_p_s = a->min_p_all;
  p.token = reinterpret_cast<long long*>(a->token);
  p.logprob = a->logprob;
  p.V = a->V;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(a->B);
  if (a->dtype == KATA_DTYPE_BF16)
    sample_kernel<__nv_bfloat16><<<grid, kST, 0, st>>>(p);
  else if (a->dtype == KATA_DTYPE_F16)
    sample_kernel<__half><<<grid, kST, 0, st>>>(p);
  else
    sample_kernel<float><<<grid, kST, 0, st>>>(p);
  return from_cuda(cudaGetLastError());
}
