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
// p Z_k).
//   top-k: the k-th largest of the threads' maxima (four each) is not above the k-th largest logit; a histogram of the
//   maxima (four atomics a thread, not one an element) finds it to a bin of 1/64.  When what is at least that
//   large fits a list of kList elements, it is gathered and sorted, and everything after it happens on the list.
//   top-p: a pass sums all masses to Z.  What weighs less than (1 - p) Z / V is after the cut whatever the rest
//   is; the others are counted by bins of the exponent, 1/128 wide (the atomics of a full histogram took three
//   quarters of a large batch's time), and counts times the bins' middles say nearly where the cut is.  A second pass sums what lies before the bins around it, which the
//   draw needs anyway, and gathers those bins: whether the cut is among them is then known exactly, and if so
//   the sorted list has it.  (Exact masses in a histogram cost two atomics a token, one with its result.)
//   Where a list overflows (thousands of equal logits at the cut, as 16-bit types have) or misses, the cut is
//   found by digits instead: histograms of the distance, then of the bits of the logit and of the index, each within
//   the bin of the one before.
//
// A cluster of up to 8 CTAs shares a row (fewer with more rows), each keeping its part in shared memory where it
// fits, so that HBM is read once.  Where it does not (256 x 131072: 192 KB and more a CTA), later passes read it
// again, from L2 as far as the batch fits there.  Histograms are merged, and lists and sums
// gathered in the first CTA, through distributed shared memory.  A call of one row is bound by the latency
// of these steps, a large batch by the instructions of its passes, the exponentials first.
//
// Measured (device time): 1 x 32000 top-k and top-p 16 us; 64 x 32000 fp32, temperature only, 13.5 us; 1 x 131072
// nucleus 49 us; 256 x 131072 bf16 plain 62 us, top-k 47 us, nucleus 223 us, settings by row 248 us (10.4 us for the
// bytes), fp32 plain 66 us, nucleus 218 us (20.8 us for the bytes).
#include <algorithm>
#include <cmath>

#include "attn_common.cuh"
#include "host_util.h"
#include "kata_b200.h"
#include "sm100.cuh"

namespace kata {
namespace {

constexpr int kST = 512;  // threads per CTA
constexpr int kSW = kST / 32;
constexpr int kBins = 2048;
constexpr int kList = 2048;          // elements sorted directly
constexpr int kFine = 2 * kBins;     // bins of the exponent
constexpr int kChunks = 8 * kSW;     // warps of a row
constexpr int kTile = 256;           // elements a warp takes at once: 8 a lane
constexpr int kMaxV = 1 << 22;       // find_cut has 22 bits of the index, from_list packs as many beside a mass
constexpr int kStage = 96 * 1024;    // bytes of a part of a row that are kept in shared memory
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
  int cs;      // CTAs a row
  int seg;     // elements a CTA takes, a multiple of kSW kTile
  int staged;  // whether they are kept in shared memory
};

// The order of tokens as ascending numbers: the bits of -x as an unsigned number (-0 counts as 0), then the index
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  const uint32_t k = ~key;
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ u64 order_of(float x, int i) { return static_cast<u64>(order_key(x)) << 32 | static_cast<uint32_t>(i); }

struct Row {
  float m, inv;  // maximum, 1 / temperature
  bool odd;      // an infinite maximum or temperature
  // A mask weighs nothing even at an infinite temperature, nor does anything beside an infinite logit.  Otherwise
  // exp gives both by itself.
  __device__ __forceinline__ float z(float x) const { return odd && x == m ? 0.f : __fmul_rn(__fsub_rn(x, m), inv); }
  __device__ __forceinline__ float w(float x) const {
    if (odd) return x == m ? 1.f : (x == -INFINITY || m == INFINITY) ? 0.f : expf(z(x));
    return expf(z(x));
  }
  // Whole numbers growing with the distance from the maximum: adding 2^23 rounds to one and leaves it in the low bits
  __device__ __forceinline__ static uint32_t whole(float t, int last) {
    return __float_as_uint(__fadd_rn(fminf(t, static_cast<float>(last)), 8388608.f)) - 0x4b000000u;
  }
  __device__ __forceinline__ uint32_t bin(float x) const {
    return odd && x == m ? 0u : whole(__fmul_rn(__fsub_rn(m, x), 64.f), kBins - 1);
  }
  __device__ __forceinline__ uint32_t fine(float x, float z) const {  // an infinitely distant mask's 0 * inf is not a number
    return odd && !(z <= 0.f) ? kFine - 1u : whole(__fmul_rn(z, -128.f), kFine - 1);
  }
};
// rint(w 2^40) for w in [0, 1], in two parts of 20 bits: adding 1.5 2^23 rounds to a whole number and leaves it
// in the low bits (the conversion to 64 bits runs at a sixteenth of the rate)
__device__ __forceinline__ void mass_parts(float w, int& hi, int& lo) {
  const float magic = 12582912.f;
  const float t = w * 1048576.f, h = __fadd_rn(t, magic);
  const float l = __fmaf_rn(__fsub_rn(t, __fsub_rn(h, magic)), 1048576.f, magic);
  hi = __float_as_int(h) - 0x4b400000;
  lo = __float_as_int(l) - 0x4b400000;
}
__device__ __forceinline__ u64 mass_of(float w) {
  int hi, lo;
  mass_parts(w, hi, lo);
  return static_cast<u64>((static_cast<long long>(hi) << 20) + lo);
}

struct alignas(16) Smem {  // the part of the row follows it, in 16-byte vectors
  uint32_t cnt[kFine];           // a histogram of counts; of masses, low words and from kBins on the high ones
  u64 list[kList];               // first CTA
  u64 keep[kChunks], sure[kChunks];  // first CTA: of each warp of the row, what it keeps and what lies before the cut
  u64 wsum[kSW], scan[kSW];
  u64 part, part2;               // what this CTA tells the others
  u64 before, cut, total;
  uint32_t n_list, bin, bin_hi, n_bin;
};

__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ uint32_t remote(const void* p, int rank) { return mapa_shared(smem_u32(p), rank); }
// Without a memory clobber, so that several are in flight at once (one takes 600 cycles); the barriers around
// them are volatile too and keep their places.
__device__ __forceinline__ uint32_t ld32_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ u64 ld64_cluster(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st32_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st64_cluster(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
// total * n24 / 2^24, rounded down or up
__device__ __forceinline__ u64 share(u64 total, u64 n24, bool up) {
  const u64 hi = __umul64hi(total, n24), lo = total * n24;
  return (hi << 40) + (lo >> 24) + ((up && (lo & 0xffffffull)) ? 1 : 0);
}

// The digit of a place in a range of width + 1: (place - first) >> shift is below kBins, and eight neighbours share one
__host__ __device__ constexpr int index_shift(uint32_t width) {
  int shift = 3;
  while (width >> shift >= kBins) ++shift;
  return shift;
}
// Two digits leave no more places than the list holds, whatever the row's length and alignment
static_assert((1 << index_shift((1u << index_shift(kMaxV + 7)) - 1)) <= kList, "digits of places");

// Ascending sort of n different numbers by the CTA.  Up to one a thread: each finds its rank (8 cycles a number);
// beyond that by merging (66 steps of 300 cycles for 2048).
__device__ __noinline__ void sort_list(u64* list, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= kST) {
    const u64 mine = tid < n ? list[tid] : 0;
    int rank = 0;
    if (tid < (n + 31) / 32 * 32) {
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += list[j] < mine;
    }
    __syncthreads();
    if (tid < n) list[rank] = mine;
    __syncthreads();
    return;
  }
  int size = 1024;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kST) list[i] = ~0ull;
  for (int k = 2; k <= size; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      // within 64 numbers a warp's pairs are its own
      if (j >= 32 || k <= 2)
        __syncthreads();
      else
        __syncwarp();
      for (int i = tid; i < size / 2; i += kST) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const u64 va = list[a], vb = list[b];
        if ((va > vb) == ((a & k) == 0)) {
          list[a] = vb;
          list[b] = va;
        }
      }
    }
  }
  __syncthreads();
}

template <typename T>
struct Sampler {
  const SampleParams& p;
  Smem& s;
  T* stage;
  const T* x;      // the row
  int rank, tid, lane, warp;
  int skew;        // places count from the 16-byte boundary at or before the row: place = index + skew
  int lo;          // this CTA's first place
  Row row;

  // A word of each CTA of the row (0 past them), lane by lane
  __device__ __forceinline__ u64 of_all(const u64* w) const { return lane < p.cs ? ld64_cluster(remote(w, lane)) : 0; }
  __device__ __forceinline__ static u64 sum32(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  __device__ __forceinline__ void sync() const {
    __syncwarp();  // the cluster barrier is one instruction for a warp
    if (p.cs > 1)
      cluster_sync();
    else
      __syncthreads();
  }
  // The eight logits from place e (a multiple of 8) as they lie; -inf outside the row
  struct alignas(16) Eight {
    T t[8];
    __device__ __forceinline__ float operator[](int j) const { return fmaxf(to_f32<T>(t[j]), -INFINITY); }  // NaN: -inf
  };
  __device__ __forceinline__ Eight load_edge(int e) const {
    Eight r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.t[j] = e + j >= skew && e + j < skew + p.V ? x[e + j - skew] : from_f32<T>(-INFINITY);
    return r;
  }
  __device__ __forceinline__ Eight load(int e) const {
    if (e < skew || e + 8 > skew + p.V) return load_edge(e);
    Eight r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
      reinterpret_cast<uint4*>(r.t)[i] = __ldg(reinterpret_cast<const uint4*>(x + (e - skew)) + i);
    return r;
  }
  __device__ __forceinline__ float one(int e) const {  // the logit of a place
    if (p.staged) return fmaxf(to_f32<T>(stage[e - lo]), -INFINITY);
    return e >= skew && e < skew + p.V ? fmaxf(to_f32<T>(x[e - skew]), -INFINITY) : -INFINITY;
  }
  __device__ __forceinline__ Eight get(int e) const {
    if (!p.staged) return load(e);
    Eight r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(r.t)[i] = reinterpret_cast<const uint4*>(stage + (e - lo))[i];
    return r;
  }
  __device__ __forceinline__ static float max8(const Eight& r) {
    float m;
    if constexpr (sizeof(T) == 4) {
      m = r[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) m = fmaxf(m, r[j]);
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* q = reinterpret_cast<const T2*>(r.t);
      const T2 a = __hmax2(__hmax2(q[0], q[1]), __hmax2(q[2], q[3]));  // a number where there is one
      m = fmaxf(fmaxf(to_f32<T>(a.x), to_f32<T>(a.y)), -INFINITY);
    }
    return m;
  }
  // f(eight logits, place) over the places [a, b), for a warp; whole tiles
  template <typename F>
  __device__ __forceinline__ void each8(int a, int b, F f) const {
    if (a >= b) return;
    Eight next = get(a + lane * 8);
    for (int e = a + lane * 8; e < b; e += kTile) {
      const Eight r = next;
      if (e + kTile < b) next = get(e + kTile);  // on its way while this one is worked on
      f(r, e);
    }
  }
  // f(logit, index) over those with a logit of at least `floor` among their eight
  template <typename F>
  __device__ __forceinline__ void each(int a, int b, float floor, F f) const {
    each8(a, b, [&](const Eight& r, int e) {
      if (__any_sync(0xffffffffu, max8(r) >= floor)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f(r[j], e + j - skew);
      }
    });
  }
  __device__ __forceinline__ int warp_lo() const { return lo + warp * (p.seg / kSW); }
  __device__ __forceinline__ int warp_hi() const { return min(warp_lo() + p.seg / kSW, (skew + p.V + kTile - 1) / kTile * kTile); }

  // Inclusive sums of 4 values a thread over the CTA, as the sum before the thread's first one
  __device__ __forceinline__ u64 block_before(u64 mine, u64* total) {
    const u64 inc = warp_scan(mine, lane);
    __syncthreads();
    if (lane == 31) s.scan[warp] = inc;
    __syncthreads();
    u64 base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSW; ++w) {
      if (w < warp) base += s.scan[w];
      all += s.scan[w];
    }
    *total = all;
    return base + inc - mine;
  }

  // The bin of the whole row's histogram where the inclusive sum reaches rem: s.bin, s.before, s.n_bin everywhere;
  // false when it does not
  template <bool BY_MASS>
  __device__ __forceinline__ bool find_bin(u64 rem) {
    sync();  // histograms are complete
    const int per = kBins / p.cs, first = rank * per;  // this CTA's bins; 4 a thread at most
    u64 v[4] = {0, 0, 0, 0}, sum = 0;
    const int mine = per / kST > 0 ? per / kST : 1;
    const int b0 = first + tid * mine;
    if (tid * mine < per) {
      for (int j = 0; j < mine; ++j) {
        u64 t = 0;
        if (p.cs == 1) {
          t = s.cnt[b0 + j] + (BY_MASS ? static_cast<u64>(s.cnt[kBins + b0 + j]) << 32 : 0);
        } else {
          uint32_t l[8], h[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            l[c] = c < p.cs ? ld32_cluster(remote(&s.cnt[b0 + j], c)) : 0;
            h[c] = BY_MASS && c < p.cs ? ld32_cluster(remote(&s.cnt[kBins + b0 + j], c)) : 0;
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) t += l[c] + (static_cast<u64>(h[c]) << 32);
        }
        v[j] = t;
        sum += t;
      }
    }
    u64 total;
    u64 before = block_before(sum, &total);
    if (p.cs > 1) {
      if (tid == 0) s.part = total;
      cluster_sync();
      const u64 t = of_all(&s.part);
      before += sum32(lane < rank ? t : 0);
      total = sum32(t);
    }
    for (int j = 0; j < mine; ++j) {
      if (before < rem && before + v[j] >= rem) {
        for (int c = 0; c < p.cs; ++c) {
          st32_cluster(remote(&s.bin, c), b0 + j);
          st64_cluster(remote(&s.before, c), before);
          st32_cluster(remote(&s.n_bin, c), BY_MASS ? 0u : static_cast<uint32_t>(v[j]));
        }
      }
      before += v[j];
    }
    sync();
    return total >= rem;
  }

  // The first and last bin of the exponent that may well hold the element where the mass reaches rem: s.bin, s.bin_hi
  // everywhere.  A bin's mass is taken as its count times its middle's, give or take a thousandth.
  __device__ __forceinline__ void find_range(u64 rem) {
    sync();  // histograms are complete
    const int per = kFine / p.cs, mine = per / kST;  // 1 to 8 bins a thread
    const int b0 = rank * per + tid * mine;
    u64 low = 0, high = 0;
    uint32_t n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      n[j] = 0;
      if (j < mine) {
        if (p.cs == 1) {
          n[j] = s.cnt[b0 + j];
        } else {
          uint32_t t[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) t[c] = c < p.cs ? ld32_cluster(remote(&s.cnt[b0 + j], c)) : 0;
#pragma unroll
          for (int c = 0; c < 8; ++c) n[j] += t[c];
        }
        high += n[j] * most(b0 + j);
        low += n[j] * least(b0 + j);
      }
    }
    u64 all_low, all_high;
    low = block_before(low, &all_low);
    high = block_before(high, &all_high);
    if (tid == 0) s.bin = s.bin_hi = kFine - 1;
    if (p.cs > 1) {
      if (tid == 0) {
        s.part = all_low;
        s.part2 = all_high;
      }
      cluster_sync();
      const u64 l = of_all(&s.part), h = of_all(&s.part2);
      low += sum32(lane < rank ? l : 0);
      high += sum32(lane < rank ? h : 0);
    } else {
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= mine) break;
      const u64 dl = n[j] * least(b0 + j), dh = n[j] * most(b0 + j);
      if (high < rem && high + dh >= rem)
        for (int c = 0; c < p.cs; ++c) st32_cluster(remote(&s.bin, c), b0 + j);
      if (low < rem && low + dl >= rem)
        for (int c = 0; c < p.cs; ++c) st32_cluster(remote(&s.bin_hi, c), b0 + j);
      low += dl;
      high += dh;
    }
    sync();
  }
  __device__ __forceinline__ static u64 most(int b) {
    return static_cast<u64>(exp2f(b * (-1.44269504f / 128)) * (1.001f * 1099511627776.f)) + 1;
  }
  __device__ __forceinline__ static u64 least(int b) {
    return b == kFine - 1 ? 0 : static_cast<u64>(exp2f(b * (-1.44269504f / 128)) * (0.999f * 1099511627776.f));
  }

  // Appends to this CTA's list
  __device__ __forceinline__ void append(bool yes, float v, int i) {
    if (!yes || *static_cast<volatile uint32_t*>(&s.n_list) > kList) return;  // too many: no more of them queue up
    const uint32_t at = atomicAdd(&s.n_list, 1u);
    if (at < kList) s.list[at] = order_of(v, i);
  }
  // The CTAs' lists (complete, and a barrier since) to the first one's; returns how many there are: more than kList
  // are not collected
  __device__ __forceinline__ uint32_t collect() {
    if (p.cs == 1) return s.n_list;
    const uint32_t mine = s.n_list, n = lane < p.cs ? ld32_cluster(remote(&s.n_list, lane)) : 0;
    const uint32_t all = __reduce_add_sync(0xffffffffu, n), before = __reduce_add_sync(0xffffffffu, lane < rank ? n : 0);
    if (all <= kList && rank > 0)
      for (uint32_t i = tid; i < mine; i += kST) st64_cluster(remote(&s.list[before + i], 0), s.list[i]);
    sync();
    return all;
  }
  // A logit that every one of the first `b` bins of the distance is above
  __device__ __forceinline__ float floor_of(uint32_t b) const {
    return row.odd || b >= kBins - 1 ? -INFINITY : __fsub_rn(row.m, (b + 2) * (1.f / 64)) - fabsf(row.m) * 1e-6f;
  }

  // Sorts the list (first CTA) and finds where its inclusive sum reaches rem: s.cut; false when it does not
  template <bool BY_MASS>
  __device__ __forceinline__ bool cut_in_list(int n, u64 rem) {
    sort_list(s.list, n);
    u64 q[4], sum = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * 4 + j;
      q[j] = i >= n ? 0 : BY_MASS ? mass_of(row.w(key_value(static_cast<uint32_t>(s.list[i] >> 32)))) : 1;
      sum += q[j];
    }
    u64 b = block_before(sum, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (b < rem && b + q[j] >= rem) s.cut = s.list[tid * 4 + j];
      b += q[j];
    }
    __syncthreads();
    return total >= rem;
  }

  // The beginning of the order, the first k at least, as the first CTA's sorted list, by way of the threads' maxima;
  // false when these are too few or the list overflows
  __device__ __forceinline__ bool list_top(int k, const float (&tops)[4]) {
    if (k > p.cs * kST * 2) return false;
    for (int i = tid; i < kBins; i += kST) s.cnt[i] = 0;
    if (tid == 0) s.n_list = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tops[j] > -INFINITY) atomicAdd(&s.cnt[row.bin(tops[j])], 1u);
    if (!find_bin<false>(k)) return false;
    const uint32_t b1 = s.bin;
    each(warp_lo(), warp_hi(), floor_of(b1), [&](float v, int i) { append(v > -INFINITY && row.bin(v) <= b1, v, i); });
    sync();
    const uint32_t n = collect();
    if (n <= kList && rank == 0) sort_list(s.list, n);
    sync();  // everybody has read the list's length
    return n <= kList;
  }

  // Finds the first token of the order whose inclusive count (BY_MASS: inclusive mass) is at least `limit`,
  // which the row's total reaches: s.cut everywhere.  With BY_MASS false, true when instead the first CTA's
  // list holds the whole beginning of the order up to the cut (and a little more), sorted: s.n_list of it.
  template <bool BY_MASS>
  __device__ bool find_cut(u64 limit) {
    int b1 = -1;
    u64 prefix = 0, mask = 0, rem = limit;
    for (int level = 0;; ++level) {
      // digits in turn: distance bin, key bits (11, 11, 10), index bits (11, 11)
      const int shift = level == 1 ? 53 : level == 2 ? 42 : level == 3 ? 32 : level == 4 ? 11 : 0;
      const uint32_t width = level == 3 ? 1023u : 2047u;
      for (int i = tid; i < kBins; i += kST) s.cnt[i] = s.cnt[kBins + i] = 0;
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      each(warp_lo(), warp_hi(), b1 < 0 ? -INFINITY : floor_of(b1), [&](float v, int i) {
        if (v == -INFINITY) return;
        uint32_t d = row.bin(v);
        if (level > 0) {
          const u64 o = order_of(v, i);
          if (static_cast<int>(d) != b1 || ((o ^ prefix) & mask)) return;
          d = static_cast<uint32_t>(o >> shift) & width;
        }
        if (BY_MASS) {
          const u64 q = mass_of(row.w(v));
          if (q == 0) return;
          const uint32_t ql = static_cast<uint32_t>(q), old = atomicAdd(&s.cnt[d], ql);
          const uint32_t qh = static_cast<uint32_t>(q >> 32) + (old + ql < old ? 1u : 0u);
          if (qh) atomicAdd(&s.cnt[kBins + d], qh);
        } else {
          atomicAdd(&s.cnt[d], 1u);
        }
      });
      // masked tokens end the order and have no mass: with fewer than k others nothing is cut
      if (!find_bin<BY_MASS>(rem)) {
        s.cut = ~0ull;
        __syncthreads();
        return false;
      }
      const uint32_t d = s.bin;
      const u64 before = s.before;
      const uint32_t n_bin = s.n_bin;
      rem -= before;
      if (level == 0) {
        b1 = d;
        if (!BY_MASS && before + n_bin <= kList) {
          each(warp_lo(), warp_hi(), floor_of(b1),
               [&](float v, int i) { append(v > -INFINITY && row.bin(v) <= static_cast<uint32_t>(b1), v, i); });
          sync();
          const uint32_t n_all = collect();
          if (rank == 0) sort_list(s.list, n_all);
          return true;
        }
      } else {
        prefix |= static_cast<u64>(d) << shift;
        mask |= static_cast<u64>(width) << shift;
      }
      if (BY_MASS || n_bin <= kList) {
        each(warp_lo(), warp_hi(), floor_of(b1), [&](float v, int i) {
          append(v > -INFINITY && static_cast<int>(row.bin(v)) == b1 && ((order_of(v, i) ^ prefix) & mask) == 0, v, i);
        });
        sync();
        const uint32_t n = collect();
        if (n <= kList) {
          if (rank == 0) cut_in_list<BY_MASS>(n, rem);
          sync();
          const u64 cut = p.cs > 1 ? ld64_cluster(remote(&s.cut, 0)) : s.cut;
          sync();
          if (tid == 0) s.cut = cut;
          __syncthreads();
          return false;
        }
      }
      sync();  // everybody has read the list's length
    }
  }

  // The cut by mass among the elements in the exponent's bins b_lo..b_hi (logits of `floor` at least), by the digits of
  // their keys, counted from the range's first one, and where equal logits are too many, of their indexes: s.cut
  // everywhere; false when their mass does not reach rem
  __device__ __forceinline__ bool cut_in_range(u64 rem, uint32_t b_lo, uint32_t b_hi, float floor) {
    // a logit above all of the range: the slack of `above` the other way
    const float ceil = row.odd || b_lo < 3 ? INFINITY : __fsub_rn(row.m, (b_lo - 2) * (1.f / 128) / row.inv) + fabsf(row.m) * 1e-6f;
    uint32_t key = order_key(ceil), span = order_key(floor) - key;    // keys key .. key + span
    uint32_t place = 0, width = static_cast<uint32_t>(p.V + skew - 1);  // places place .. place + width
    uint32_t* count = reinterpret_cast<uint32_t*>(s.list);
    // Each round takes a digit of the keys, or once one is left, of the places, and narrows their range to the digit's:
    // three of the keys at most, and two of the places, since V <= kMaxV and a digit of the lowest three bits, eight
    // neighbours, always fits the list.
    for (;;) {
      const bool by_index = span == 0;
      const int shift = by_index ? index_shift(width) : max(0, 21 - __clz(span));  // span >> shift < 2048
      auto in = [&](float v, int i) {
        const uint32_t d = row.fine(v, row.z(v));
        return v >= floor && v > -INFINITY && d >= b_lo && d <= b_hi && order_key(v) - key <= span && i + skew - place <= width;
      };
      for (int i = tid; i < kBins; i += kST) s.cnt[i] = s.cnt[kBins + i] = count[i] = 0;
      __syncthreads();
      auto add = [&](uint32_t d, u64 q, uint32_t n) {
        const uint32_t ql = static_cast<uint32_t>(q), old = atomicAdd(&s.cnt[d], ql);
        const uint32_t qh = static_cast<uint32_t>(q >> 32) + (old + ql < old ? 1u : 0u);
        if (qh) atomicAdd(&s.cnt[kBins + d], qh);
        atomicAdd(&count[d], n);
      };
      if (by_index) {  // one logit: a thread's eight neighbours at once
        const u64 q = mass_of(row.w(key_value(key)));
        each8(warp_lo(), warp_hi(), [&](const Eight& r, int e) {
          if (!(max8(r) >= floor)) return;
          uint32_t n = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) n += in(r[j], e + j - skew);
          if (n) add((e - place) >> shift, n * q, n);
        });
      } else {
        each(warp_lo(), warp_hi(), floor, [&](float v, int i) {
          if (in(v, i)) add((order_key(v) - key) >> shift, mass_of(row.w(v)), 1);
        });
      }
      if (!find_bin<true>(rem)) return false;
      rem -= s.before;
      const uint32_t d = s.bin;
      const uint32_t n_bin = __reduce_add_sync(0xffffffffu, lane < p.cs ? ld32_cluster(remote(&count[d], lane)) : 0);
      if (by_index) {
        place += d << shift;
        width = (1u << shift) - 1;
      } else {
        key += d << shift;
        span = (1u << shift) - 1;
      }
      sync();  // everybody has read the counts, which share the list's memory
      if (n_bin > kList) continue;
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      each(warp_lo(), warp_hi(), floor, [&](float v, int i) { append(in(v, i), v, i); });
      sync();
      const uint32_t n = collect();
      if (rank == 0) cut_in_list<true>(n, rem);
      sync();
      const u64 cut = p.cs > 1 ? ld64_cluster(remote(&s.cut, 0)) : s.cut;
      sync();
      if (tid == 0) s.cut = cut;
      __syncthreads();
      return true;
    }
  }

  __device__ void answer(long long b, int i, u64 total, bool greedy) const {
    const float v = to_f32<T>(x[i]);
    p.token[b] = i;
    p.logprob[b] = greedy ? 0.f : row.z(v) - static_cast<float>(log(static_cast<double>(total) * 0x1p-40));
  }

  __device__ void run(long long b) {
    const float temp = p.temperature ? p.temperature[b] : p.temperature_s;
    const float top_p = p.top_p ? p.top_p[b] : p.top_p_s;
    const float min_p = p.min_p ? p.min_p[b] : p.min_p_s;
    int k = p.top_k ? p.top_k[b] : p.top_k_s;
    const float uu = p.u[b];
    const u64 p24 = top_p > 0.f ? static_cast<u64>(fminf(top_p, 1.f) * 16777216.f) : 0;
    if (k <= 0 || k > p.V) k = p.V;
    if (!(temp > 0.f) || min_p > 1.f || p24 == 0) k = 1;  // only the first token is kept
    u64 u24 = uu > 0.f ? static_cast<u64>(fminf(uu, 1.f) * 16777216.f) : 0;
    if (u24 > 16777215ull) u24 = 16777215ull;

    // The first token of the order; the row's part into shared memory
    u64 first = ~0ull;
    float best = -INFINITY;
    int best_e = 0;
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // maxima of a quarter of the thread's elements each
    const int hi_e = warp_hi(), e_lo = warp_lo() + lane * 8;
    auto take = [&](const Eight& r, int e, bool before) {
      if (p.staged) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(stage + (e - lo))[i] = reinterpret_cast<const uint4*>(r.t)[i];
      }
      const float m = max8(r);
      if (m > best || (before && m == best)) {
        best = m;
        best_e = e;
      }
      return m;
    };
    constexpr int AHEAD = sizeof(T) == 2 ? 8 : 4;  // loads in flight: the pass over HBM
#pragma unroll 1
    for (int e0 = e_lo; e0 < hi_e; e0 += AHEAD * kTile) {
      Eight r[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int e = e0 + u * kTile;
        if (e < hi_e && e >= skew && e + 8 <= skew + p.V) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            reinterpret_cast<uint4*>(r[u].t)[i] = __ldg(reinterpret_cast<const uint4*>(x + (e - skew)) + i);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) r[u].t[j] = from_f32<T>(-INFINITY);
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (e0 + u * kTile < hi_e) tops[u & 3] = fmaxf(tops[u & 3], take(r[u], e0 + u * kTile, false));
      }
    }
    // the row's first and last eight, where they are not whole
#pragma unroll 1
    for (int end = 0; end < 2; ++end) {
      const int e = end ? (skew + p.V) / 8 * 8 : 0;
      const bool whole = end ? (skew + p.V) % 8 == 0 || (e == 0 && skew > 0) : skew == 0;
      if (!whole && e >= e_lo && e < hi_e && (e - e_lo) % kTile == 0) tops[0] = fmaxf(tops[0], take(load_edge(e), e, end == 0));
    }
    // where it is, from the threads that have the CTA's largest
    float m = best;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s.scan[warp] = __float_as_uint(m);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSW; ++w) m = fmaxf(m, __uint_as_float(static_cast<uint32_t>(s.scan[w])));
    if (best == m && m > -INFINITY) {
#pragma unroll 1
      for (int j = 7; j >= 0; --j)
        if (one(best_e + j) == best) first = order_of(best, best_e + j - skew);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    if (lane == 0) s.wsum[warp] = first;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSW; ++w) first = min(first, s.wsum[w]);
    if (p.cs > 1) {
      if (tid == 0) s.part = first;
      cluster_sync();
      if (lane < p.cs) first = ld64_cluster(remote(&s.part, lane));
#pragma unroll
      for (int o = 16; o; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      cluster_sync();
    }
    if (first == ~0ull) {  // nothing to draw from
      if (rank == 0 && tid == 0) {
        p.token[b] = -1;
        p.logprob[b] = -INFINITY;
      }
      return;
    }
    if (k == 1) {
      if (rank == 0 && tid == 0) answer(b, static_cast<int>(first & 0xffffffffu), 0, true);
      return;
    }
    row.m = key_value(static_cast<uint32_t>(first >> 32));
    row.inv = 1.f / temp;
    row.odd = row.m == INFINITY || row.inv == 0.f || row.inv == INFINITY;

    u64 cut = ~0ull;
    if (k < p.V) {
      if (list_top(k, tops) || find_cut<false>(k)) {
        if (rank == 0) from_list(b, k, top_p, p24, min_p, u24);
        sync();
        return;
      }
      cut = s.cut;
    }
    if (top_p < 1.f) {
      // all masses
      u64 t = 0;
      const bool has_cut = cut != ~0ull;
      const float cut_v = key_value(static_cast<uint32_t>(cut >> 32));
      if (cut == ~0ull && !row.odd)
        t = masses(0.f);
      else
        each(warp_lo(), warp_hi(), -INFINITY, [&](float v, int i) { t += kept(v, i, cut, 0.f); });
      const u64 z_mass = total_of(t), limit = share(z_mass, p24, true);
      // the counts of the exponent's bins, down to a weight of (1 - p) Z / V
      for (int i = tid; i < kBins; i += kST) s.cnt[i] = s.cnt[kBins + i] = 0;
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      const float least_w = static_cast<float>(z_mass - limit) * (0.99f / 1099511627776.f) / static_cast<float>(p.V);
      const uint32_t b_end = row.odd ? kFine - 1 : whole_bins(least_w);
      const float bulk = row.odd || b_end >= kFine - 1 ? -INFINITY : above(b_end);
      each8(warp_lo(), warp_hi(), [&](const Eight& r, int e) {
        if (!(max8(r) >= bulk)) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = r[j];
          if (!(v >= bulk) || v == -INFINITY) continue;
          if (has_cut && (v < cut_v || (v == cut_v && order_of(v, e + j - skew) > cut))) continue;
          atomicAdd(&s.cnt[row.fine(v, row.z(v))], 1u);
        }
      });
      find_range(limit);
      const uint32_t b_lo = s.bin, b_hi = s.bin_hi;
      // what lies surely before the cut, and a list of what may be the cut
      const float floor = row.odd || b_hi >= kFine - 1 ? -INFINITY : above(b_hi);
      u64 sure = 0, keep = 0;
      each8(warp_lo(), warp_hi(), [&](const Eight& r, int e) {
        if (!__any_sync(0xffffffffu, max8(r) >= floor)) return;
        uint32_t maybe = 0;
        int sh = 0, sl = 0, kh = 0, kl = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // without branches: most steps have something to add
          const float v = r[j], z = row.z(v), w = row.odd ? row.w(v) : expf(z);
          bool in = v > -INFINITY;
          if (has_cut) in = in && !(v < cut_v || (v == cut_v && order_of(v, e + j - skew) > cut));
          const uint32_t d = in ? row.fine(v, z) : kFine;
          int h, l;
          mass_parts(d < b_lo ? w : 0.f, h, l);
          sh += h;
          sl += l;
          const bool k = !(w < min_p);  // as kept()
          kh += k ? h : 0;
          kl += k ? l : 0;
          maybe |= (d >= b_lo && d <= b_hi ? 1u : 0u) << j;
        }
        sure += static_cast<u64>((static_cast<long long>(sh) << 20) + sl);
        keep += static_cast<u64>((static_cast<long long>(kh) << 20) + kl);
        if (maybe) {
#pragma unroll
          for (int j = 0; j < 8; ++j) append(maybe >> j & 1, r[j], e + j - skew);
        }
      });
      tell(keep, sure);
      const uint32_t n = collect();
      if (n <= kList) {
        if (rank == 0) {
          u64 before = 0;
#pragma unroll
          for (int c = 0; c < kChunks; c += 32) before += c + lane < p.cs * kSW ? s.sure[c + lane] : 0;
          before = sum32(before);
          const bool found = before < limit && cut_in_list<true>(n, limit - before);
          if (tid == 0) s.n_bin = found;
          for (int i = tid; found && i < static_cast<int>(n); i += kST) {
            const u64 o = s.list[i];
            const float w = row.w(key_value(static_cast<uint32_t>(o >> 32)));
            if (o <= s.cut && !(w < min_p)) atomicAdd(&s.keep[(static_cast<uint32_t>(o) + skew) / (p.seg / kSW)], mass_of(w));
          }
          __syncthreads();
        }
        if (draw(b, u24, min_p, true)) return;
        sync();
      } else {  // thousands of equal or nearly equal logits at the cut
        u64 before = 0;
#pragma unroll
        for (int c = 0; c < kChunks; c += 32) before += c + lane < p.cs * kSW ? ld64_cluster(remote(&s.sure[c + lane], 0)) : 0;
        before = sum32(before);
        sync();  // everybody has read the list's length and the sums
        if (before < limit && cut_in_range(limit - before, b_lo, b_hi, floor)) {
          cut = min(cut, s.cut);
          each(warp_lo(), warp_hi(), floor, [&](float v, int i) {
            const uint32_t d = row.fine(v, row.z(v));
            if (d >= b_lo && d <= b_hi) keep += kept(v, i, cut, min_p);
          });
          if (rank == 0 && tid == 0) s.cut = cut;
          tell(keep, 0);
          draw(b, u24, min_p, false);
          return;
        }
        sync();
      }
      find_cut<true>(limit);
      cut = min(cut, s.cut);
    }
    u64 keep = 0;
    if (cut == ~0ull && !row.odd)
      keep = masses(min_p);
    else
      each(warp_lo(), warp_hi(), -INFINITY, [&](float v, int i) { keep += kept(v, i, cut, min_p); });
    if (rank == 0 && tid == 0) s.cut = cut;
    tell(keep, 0);
    draw(b, u24, min_p, false);
  }

  // The mass of this thread's elements of the row's whole order that weigh min_p at least
  __device__ __forceinline__ u64 masses(float min_p) const {
    u64 t = 0;
    const Row rw = row;
    each8(warp_lo(), warp_hi(), [&](const Eight& r, int) {
      int hi = 0, lo8 = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = expf(__fmul_rn(__fsub_rn(r[j], rw.m), rw.inv));
        int h, l;
        mass_parts(w < min_p ? 0.f : w, h, l);
        hi += h;
        lo8 += l;
      }
      t += static_cast<u64>((static_cast<long long>(hi) << 20) + lo8);
    });
    return t;
  }
  // The bin of the exponent that holds a weight, and a logit that every one of the bins up to b is above
  __device__ __forceinline__ static uint32_t whole_bins(float w) {
    const float t = -128.f * 0.69314718f * log2f(w) + 1.f;
    return t >= kFine - 1 ? kFine - 1 : t > 0.f ? static_cast<uint32_t>(t) : 0u;
  }
  __device__ __forceinline__ float above(uint32_t b) const {
    return __fsub_rn(row.m, (b + 2) * (1.f / 128) / row.inv) - fabsf(row.m) * 1e-6f;
  }

  __device__ __forceinline__ u64 kept(float v, int i, u64 cut, float min_p) const {
    if (v == -INFINITY || order_of(v, i) > cut) return 0;
    const float w = row.w(v);
    return w < min_p ? 0 : mass_of(w);
  }

  // A warp's sums to the first CTA
  __device__ __forceinline__ void tell(u64 keep, u64 sure) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      keep += __shfl_xor_sync(0xffffffffu, keep, o);
      sure += __shfl_xor_sync(0xffffffffu, sure, o);
    }
    if (lane == 0) {
      st64_cluster(remote(&s.keep[rank * kSW + warp], 0), keep);
      st64_cluster(remote(&s.sure[rank * kSW + warp], 0), sure);
    }
    sync();
  }

  // The token, from the first CTA's s.keep and s.cut; false (`check`) when s.n_bin says that there is no cut yet
  __device__ __forceinline__ bool draw(long long b, u64 u24, float min_p, bool check) {
    if (rank == 0 && warp == 0) {
      const int n = p.cs * kSW, per = (n + 31) / 32;  // 1 to 4 chunks a lane
      u64 sum = 0;
      for (int j = 0; j < per; ++j) sum += lane * per + j < n ? s.keep[lane * per + j] : 0;
      u64 at = warp_scan(sum, lane);
      const u64 total = __shfl_sync(0xffffffffu, at, 31), target = share(total, u24, false);
      at -= sum;
      for (int j = 0; j < per; ++j) {
        const u64 q = lane * per + j < n ? s.keep[lane * per + j] : 0;
        if (at <= target && target < at + q) {
          s.bin = lane * per + j;
          s.before = at;
          s.part2 = target;
          s.total = total;
        }
        at += q;
      }
    }
    sync();
    if (check && ld32_cluster(remote(&s.n_bin, 0)) == 0) return false;
    const int chunk = ld32_cluster(remote(&s.bin, 0));
    u64 base = ld64_cluster(remote(&s.before, 0));
    const u64 target = ld64_cluster(remote(&s.part2, 0)), total = ld64_cluster(remote(&s.total, 0));
    const u64 cut = ld64_cluster(remote(&s.cut, 0));
    sync();  // nobody reads another CTA's memory any more
    if (chunk / kSW != rank) return true;
    // in this CTA's part: its warps split the chunk
    const int a = lo + chunk % kSW * (p.seg / kSW), per = (p.seg / kSW / kTile + kSW - 1) / kSW * kTile;
    const int end = min(a + p.seg / kSW, (skew + p.V + kTile - 1) / kTile * kTile);
    const int sa = min(end, a + warp * per), sb = min(end, sa + per);
    u64 q = 0;
    each(sa, sb, -INFINITY, [&](float v, int i) { q += kept(v, i, cut, min_p); });
#pragma unroll
    for (int o = 16; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    if (lane == 0) s.scan[warp] = q;
    __syncthreads();
    for (int i = 0; i < warp; ++i) base += s.scan[i];
    if (!(base <= target && target < base + q)) return true;
    for (int e = sa; e < sb; e += kTile) {
      const Eight r = get(e + lane * 8);
      u64 ms[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += ms[j] = kept(r[j], e + lane * 8 + j - skew, cut, min_p);
      u64 at = base + warp_scan(sum, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, at > target);
      base = __shfl_sync(0xffffffffu, at, 31);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          at -= sum;
          for (int j = 0; j < 8; ++j) {
            at += ms[j];
            if (at > target) {
              answer(b, e + lane * 8 + j - skew, total, false);
              break;
            }
          }
        }
        return true;
      }
    }
    return true;
  }

  // The row's total of what the threads have
  __device__ __forceinline__ u64 total_of(u64 mine) {
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s.wsum[warp] = mine;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kSW; ++w) all += s.wsum[w];
    if (p.cs == 1) return all;
    if (tid == 0) s.part = all;
    cluster_sync();
    all = sum32(of_all(&s.part));
    cluster_sync();
    return all;
  }

  // The rest on the sorted list (first CTA): the first k tokens are its first k
  __device__ __forceinline__ void from_list(long long b, int k, float top_p, u64 p24, float min_p, u64 u24) {
    u64 q[4], sum = 0, total;
    bool low[4];
    uint32_t idx[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * 4 + j;
      q[j] = 0;
      low[j] = false;
      idx[j] = 0xffffffffu;
      if (i < k) {
        const float w = row.w(key_value(static_cast<uint32_t>(s.list[i] >> 32)));
        idx[j] = static_cast<uint32_t>(s.list[i]);
        q[j] = mass_of(w);
        low[j] = w < min_p;
      }
      sum += q[j];
    }
    u64 before = block_before(sum, &total);
    const u64 limit = top_p < 1.f ? share(total, p24, true) : ~0ull;
    sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 was = before;
      before += q[j];
      if (was >= limit || low[j]) q[j] = 0;
      sum += q[j];
    }
    block_before(sum, &total);
    const u64 target = share(total, u24, false);
    // in vocabulary order: index in the upper bits, mass (at most 2^40) below
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tid * 4 + j < k) s.list[tid * 4 + j] = static_cast<u64>(idx[j]) << 41 | q[j];
    __syncthreads();
    sort_list(s.list, k);
    sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[j] = tid * 4 + j < k ? s.list[tid * 4 + j] & ((1ull << 41) - 1) : 0;
      sum += q[j];
    }
    u64 all;
    u64 at = block_before(sum, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at <= target && target < at + q[j]) answer(b, static_cast<int>(s.list[tid * 4 + j] >> 41), total, false);
      at += q[j];
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kST) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const long long b = blockIdx.x / p.cs;
  const T* x = static_cast<const T*>(p.logits) + b * p.ld;
  const int rank = p.cs > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int tid = threadIdx.x;
  Sampler<T> me{p, s, reinterpret_cast<T*>(raw + sizeof(Smem)), x, rank, tid, tid & 31, tid >> 5, skew, rank * p.seg, Row{0.f, 0.f, false}};
  me.run(b);
}

}  // namespace
}  // namespace kata

using namespace kata;

template <typename T>
static int launch_sample(SampleParams& p, long long B, cudaStream_t st) {
  // CTAs a row: up to two an SM, with more than a tile for each warp (1 x 131072 nucleus: 49 us on 8, 155 on one).
  // Rows of their own settings differ several times in cost, and with one CTA each the last one is waited for: long
  // ones get twice as many.  From 65536 on that is ahead with every batch (160 rows: 65536 112 against 172 us, 131072
  // 217 against 306; 75 rows: 65536 80 against 100 us), below it with some (32000: 160 rows 68 against 74 us, but 140
  // rows 72 against 66; 16384: 290 rows 82 against 69 us).  With one setting for all the rows cost the same, and the
  // CTAs beyond two an SM wait (256 x 131072 nucleus: 263 against 223 us).
  const bool differ = p.temperature || p.top_k || p.top_p || p.min_p;
  const long long room = differ && p.V >= 65536 ? 592 : 296;
  p.cs = 1;
  while (p.cs < 8 && B * p.cs * 2 <= room && p.V > p.cs * kSW * kTile) p.cs *= 2;
  const int places = p.V + 16 / static_cast<int>(sizeof(T)) - 1;
  p.seg = (places + p.cs - 1) / p.cs;
  p.seg = (p.seg + kSW * kTile - 1) / (kSW * kTile) * (kSW * kTile);
  const size_t part = static_cast<size_t>(p.seg) * sizeof(T);
  p.staged = part <= kStage;
  const size_t smem = sizeof(Smem) + (p.staged ? part : 0);
  auto kern = sample_kernel<T>;
  static std::atomic<uint64_t> allowed{0};
  if (int e = allow_smem(reinterpret_cast<const void*>(kern), static_cast<int>(sizeof(Smem)) + kStage, allowed)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B * p.cs));
  cfg.blockDim = dim3(kST);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cs;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.cs > 1 ? 1 : 0;
  return from_cuda(cudaLaunchKernelEx(&cfg, kern, p));
}

extern "C" int kata_sample(const kata_sample_args* a, kata_stream_t stream) {
  if (!a) return KATA_ERR_INVALID;
  if (a->dtype != KATA_DTYPE_F32 && a->dtype != KATA_DTYPE_BF16 && a->dtype != KATA_DTYPE_F16) return KATA_ERR_DTYPE;
  if (a->B < 0 || a->V < 1 || a->B > (1ll << 28) || a->V > kMaxV) return KATA_ERR_SHAPE;
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
  if (a->dtype == KATA_DTYPE_BF16) return launch_sample<__nv_bfloat16>(p, a->B, st);
  if (a->dtype == KATA_DTYPE_F16) return launch_sample<__half>(p, a->B, st);
  return launch_sample<float>(p, a->B, st);
}
