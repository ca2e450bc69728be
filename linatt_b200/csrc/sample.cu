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
// the bits of the logit and of the index within the bin that holds the cut, until at most kList elements
// are left, which are sorted.  After the first histogram that is nearly always so; when the whole
// beginning of the order up to top-k fits the list, everything after it happens on the list.
//
// One pass over HBM: a cluster of up to 8 CTAs shares a row (fewer with more rows), each keeping its part
// in shared memory where it fits (else it is read again, from L2).  Histograms are merged, and the list
// is gathered in the first CTA, through distributed shared memory.  A call of one row is bound by the
// latency of these steps, a large batch by the instructions of the histogram's exponentials.
#include <algorithm>
#include <cmath>
#include <cstdlib>

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
constexpr int kTile = 256;           // elements a warp takes at once: 8 a lane
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
  __device__ __forceinline__ float z(float x) const { return x == m ? 0.f : __fmul_rn(__fsub_rn(x, m), inv); }
  // a mask weighs nothing even at an infinite temperature, nor does anything beside an infinite logit
  __device__ __forceinline__ float w(float x) const {
    return x == m ? 1.f : (x == -INFINITY || m == INFINITY) ? 0.f : expf(z(x));
  }
  __device__ __forceinline__ int bin(float x) const {
    return x == m ? 0 : static_cast<int>(fminf(__fmul_rn(__fsub_rn(m, x), 64.f), static_cast<float>(kBins - 1)));
  }
};
// rint(w 2^40) for w in [0, 1], in two parts of 20 bits: adding 1.5 2^23 rounds to a whole number and leaves it
// in the low bits (the conversion to 64 bits runs at a sixteenth of the rate)
__device__ __forceinline__ u64 mass_of(float w) {
  const float magic = 12582912.f;
  const float t = w * 1048576.f, h = __fadd_rn(t, magic);
  const float l = __fadd_rn(__fmul_rn(__fsub_rn(t, __fsub_rn(h, magic)), 1048576.f), magic);
  return static_cast<u64>((static_cast<long long>(__float_as_int(h) - 0x4b400000) << 20) + (__float_as_int(l) - 0x4b400000));
}

struct alignas(16) Smem {  // the part of the row follows it, in 16-byte vectors
  uint32_t cnt[kBins];           // histogram of counts, or the low words of the masses'
  uint32_t hi[kBins];            // and their high words
  u64 list[kList];               // first CTA
  u64 wsum[kSW], scan[kSW];
  u64 part;                      // what this CTA tells the others
  u64 before, cut;
  uint32_t n_list, bin, n_bin;
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
__device__ __forceinline__ uint32_t ld32_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld64_cluster(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st32_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st64_cluster(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add32_cluster(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}

// total * n24 / 2^24, rounded down or up
__device__ __forceinline__ u64 share(u64 total, u64 n24, bool up) {
  const u64 hi = __umul64hi(total, n24), lo = total * n24;
  return (hi << 40) + (lo >> 24) + ((up && (lo & 0xffffffull)) ? 1 : 0);
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

  __device__ __forceinline__ void sync() const {
    __syncwarp();  // the cluster barrier is one instruction for a warp
    if (p.cs > 1)
      cluster_sync();
    else
      __syncthreads();
  }
  // The eight logits from place e (a multiple of 8); -inf outside the row and for NaN
  __device__ __forceinline__ void load(int e, float (&v)[8]) const {
    const T* src = x + (e - skew);
    if (e >= skew && e + 8 <= skew + p.V) {
      alignas(16) T t[8];
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        reinterpret_cast<uint4*>(t)[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = e + j >= skew && e + j < skew + p.V ? to_f32<T>(src[j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (v[j] != v[j]) v[j] = -INFINITY;
  }
  __device__ __forceinline__ void get(int e, float (&v)[8]) const {
    if (!p.staged) return load(e, v);
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(stage + (e - lo))[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(t[j]);
  }
  // f(logit, index) over the places [a, b) a lane at a time, for a warp; whole tiles
  template <typename F>
  __device__ __forceinline__ void each(int a, int b, F f) const {
    for (int e = a + lane * 8; e < b; e += kTile) {
      float v[8];
      get(e, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) f(v[j], e + j - skew);
    }
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

  // The bin of the whole row's histogram where the inclusive sum reaches rem: s.bin, s.before, s.n_bin everywhere
  template <bool BY_MASS>
  __device__ void find_bin(u64 rem) {
    sync();  // histograms are complete
    const int per = kBins / p.cs, first = rank * per;  // this CTA's bins; 4 a thread at most
    u64 v[4] = {0, 0, 0, 0}, sum = 0;
    const int mine = per / kST > 0 ? per / kST : 1;
    const int b0 = first + tid * mine;
    if (tid * mine < per) {
      for (int j = 0; j < mine; ++j) {
        u64 t = 0;
        for (int c = 0; c < p.cs; ++c) {
          if (p.cs == 1) {
            t = s.cnt[b0 + j] + (BY_MASS ? static_cast<u64>(s.hi[b0 + j]) << 32 : 0);
          } else {
            t += ld32_cluster(remote(&s.cnt[b0 + j], c));
            if (BY_MASS) t += static_cast<u64>(ld32_cluster(remote(&s.hi[b0 + j], c))) << 32;
          }
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
      for (int c = 0; c < rank; ++c) before += ld64_cluster(remote(&s.part, c));
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
  }

  // Ascending sort of the first n of the list (the first CTA alone)
  __device__ void sort_list(int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kST) s.list[i] = ~0ull;
    for (int k = 2; k <= size; k *= 2) {
      for (int j = k / 2; j > 0; j /= 2) {
        // within 64 elements a warp's pairs are its own
        if (j >= 32 || (j == 16 && k == 32) || k <= 2) __syncthreads();
        else __syncwarp();
        for (int i = tid; i < size / 2; i += kST) {
          const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
          const u64 va = s.list[a], vb = s.list[b];
          if ((va > vb) == ((a & k) == 0)) {
            s.list[a] = vb;
            s.list[b] = va;
          }
        }
      }
    }
    __syncthreads();
  }

  // Appends to the first CTA's list what `want` chooses
  template <typename F>
  __device__ void gather(F want) {
    each(warp_lo(), warp_hi(), [&](float v, int i) {
      const bool yes = v > -INFINITY && want(v, i);
      const unsigned m = __ballot_sync(0xffffffffu, yes);
      if (m) {
        const int leader = __ffs(m) - 1;
        uint32_t at = 0;
        if (lane == leader) at = add32_cluster(remote(&s.n_list, 0), __popc(m));
        at = __shfl_sync(0xffffffffu, at, leader) + __popc(m & ((1u << lane) - 1));
        if (yes && at < kList) st64_cluster(remote(&s.list[at], 0), order_of(v, i));
      }
    });
    sync();
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
      for (int i = tid; i < kBins; i += kST) s.cnt[i] = s.hi[i] = 0;
      if (tid == 0) s.n_list = 0;
      __syncthreads();
      each(warp_lo(), warp_hi(), [&](float v, int i) {
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
          if (qh) atomicAdd(&s.hi[d], qh);
        } else {
          atomicAdd(&s.cnt[d], 1u);
        }
      });
      find_bin<BY_MASS>(rem);
      const uint32_t d = s.bin;
      const u64 before = s.before;
      const uint32_t n_bin = s.n_bin;
      rem -= before;
      if (level == 0) {
        b1 = d;
        if (!BY_MASS && before + n_bin <= kList) {
          gather([&](float v, int) { return row.bin(v) <= b1; });
          if (rank == 0) sort_list(s.n_list);
          return true;
        }
      } else {
        prefix |= static_cast<u64>(d) << shift;
        mask |= static_cast<u64>(width) << shift;
      }
      if (BY_MASS || n_bin <= kList) {
        gather([&](float v, int i) { return row.bin(v) == b1 && ((order_of(v, i) ^ prefix) & mask) == 0; });
        const uint32_t n = ld32_cluster(remote(&s.n_list, 0));
        if (n <= kList) {
          if (rank == 0) {
            sort_list(n);
            u64 q[4], sum = 0, total;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int i = tid * 4 + j;
              q[j] = i >= static_cast<int>(n) ? 0 : BY_MASS ? mass_of(row.w(key_value(static_cast<uint32_t>(s.list[i] >> 32)))) : 1;
              sum += q[j];
            }
            u64 b = block_before(sum, &total);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (b < rem && b + q[j] >= rem) s.cut = s.list[tid * 4 + j];
              b += q[j];
            }
          }
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
    uint32_t live = 0;  // logits above -inf
    for (int e = warp_lo() + lane * 8; e < warp_hi(); e += kTile) {
      float v[8];
      load(e, v);
      if (p.staged) {
        alignas(16) T t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = from_f32<T>(v[j]);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(stage + (e - lo))[i] = reinterpret_cast<const uint4*>(t)[i];
      }
      float m = v[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) m = fmaxf(m, v[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) live += v[j] > -INFINITY;
      if (order_key(m) < static_cast<uint32_t>(first >> 32)) {
#pragma unroll
        for (int j = 7; j >= 0; --j)
          if (v[j] == m) first = order_of(m, e + j - skew);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) {
      s.wsum[warp] = first;
      s.scan[warp] = live;
    }
    __syncthreads();
    live = 0;
#pragma unroll
    for (int w = 0; w < kSW; ++w) {
      first = min(first, s.wsum[w]);
      live += static_cast<uint32_t>(s.scan[w]);
    }
    if (p.cs > 1) {
      if (tid == 0) {
        s.part = first;
        s.n_bin = live;
      }
      cluster_sync();
      live = 0;
      for (int c = 0; c < p.cs; ++c) {
        first = min(first, ld64_cluster(remote(&s.part, c)));
        live += ld32_cluster(remote(&s.n_bin, c));
      }
      cluster_sync();
    }
    const float m = key_value(static_cast<uint32_t>(first >> 32));
    row.m = m;
    row.inv = temp > 0.f ? 1.f / temp : 1.f;
    if (first == ~0ull || m == -INFINITY) {  // nothing to draw from
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

    u64 cut = ~0ull;
    // masked tokens end the order and have no mass: with no more than k others nothing is cut
    if (static_cast<uint32_t>(k) < live) {
      if (find_cut<false>(k)) {
        if (rank == 0) from_list(b, k, top_p, p24, min_p, u24);
        sync();
        return;
      }
      cut = s.cut;
    }
    auto kept = [&](float v, int i, bool floor) -> u64 {
      if (v == -INFINITY || order_of(v, i) > cut) return 0;
      const float w = row.w(v);
      return floor && w < min_p ? 0 : mass_of(w);
    };
    if (top_p < 1.f) {
      u64 t = 0;
      each(warp_lo(), warp_hi(), [&](float v, int i) { t += kept(v, i, false); });
      const u64 limit = share(total_of(t), p24, true);
      find_cut<true>(limit);
      cut = min(cut, s.cut);
    }
    u64 t = 0;
    each(warp_lo(), warp_hi(), [&](float v, int i) { t += kept(v, i, true); });
    u64 cta;
    const u64 total = total_of(t, &cta);
    const u64 target = share(total, u24, false);
    u64 base = 0;
    for (int c = 0; c < rank; ++c) base += ld64_cluster(remote(&s.part, c));
    if (base <= target && target < base + cta) {  // the token is in this CTA's part: in which warp's?
      int w = 0;
      while (target >= base + s.wsum[w]) base += s.wsum[w++];
      const int a = lo + w * (p.seg / kSW), per = (p.seg / kSW / kTile + kSW - 1) / kSW * kTile;
      const int end = min(a + p.seg / kSW, (skew + p.V + kTile - 1) / kTile * kTile);
      const int sa = min(end, a + warp * per), sb = min(end, sa + per);
      u64 q = 0;
      each(sa, sb, [&](float v, int i) { q += kept(v, i, true); });
#pragma unroll
      for (int o = 16; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      if (lane == 0) s.scan[warp] = q;
      __syncthreads();
      for (int i = 0; i < warp; ++i) base += s.scan[i];
      if (base <= target && target < base + q) {
        for (int e = sa; e < sb; e += kTile) {
          float v[8];
          get(e + lane * 8, v);
          u64 ms[8], sum = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += ms[j] = kept(v[j], e + lane * 8 + j - skew, true);
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
            break;
          }
        }
      }
    }
    sync();  // nobody reads this CTA's sums any more
  }

  // The row's total of what the threads have, and the CTA's (s.wsum of its warps, s.part for the others)
  __device__ u64 total_of(u64 mine, u64* cta = nullptr) {
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) s.wsum[warp] = mine;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < kSW; ++w) all += s.wsum[w];
    if (cta) *cta = all;
    if (p.cs == 1) return all;
    if (tid == 0) s.part = all;
    cluster_sync();
    all = 0;
    for (int c = 0; c < p.cs; ++c) all += ld64_cluster(remote(&s.part, c));
    if (!cta) cluster_sync();  // with `cta` the parts are read again
    return all;
  }

  // The rest on the sorted list (first CTA): the first k tokens are its first k
  __device__ void from_list(long long b, int k, float top_p, u64 p24, float min_p, u64 u24) {
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
    sort_list(k);
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
  Sampler<T> me{p, s, reinterpret_cast<T*>(raw + sizeof(Smem)), x, rank, tid, tid & 31, tid >> 5, skew, rank * p.seg, Row{0.f, 0.f}};
  me.run(b);
}

}  // namespace
}  // namespace kata

using namespace kata;

template <typename T>
static int launch_sample(SampleParams& p, long long B, cudaStream_t st) {
  // CTAs a row: enough to fill the GPU twice, with no fewer than two tiles a warp
  p.cs = 1;
  static const int cap = getenv("SCS") ? atoi(getenv("SCS")) : 8;
  while (p.cs < cap && B * p.cs * 2 <= 296 && p.V > p.cs * kSW * kTile) p.cs *= 2;
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
  if (a->B < 0 || a->V < 1 || a->B > (1ll << 28) || a->V > (1 << 22)) return KATA_ERR_SHAPE;
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
