// qkv_step.cu -- one token's way from the fused q/k/v projection to the recurrent attention step:
//   a[c] = sum_{j<K} w[c,j] x_{p-K+1+j}[c],  y = silu(a)            causal short convolution (K <= 4)
//   q, k heads: y / sqrt(sum y^2 + eps) or y rsqrt(mean y^2 + eps) w     norm of each head
//   q, k heads: rotation by the position's angles                        (as kata_rownorm_*)
// The K - 1 earlier inputs of a sequence are a ring: input p lies in slot p % (K - 1), so a step reads
// the whole ring and overwrites only the oldest slot.
//
// HBM-bound: (K + 1) reads and writes of a row of inputs and one of outputs.  A thread owns eight
// neighbouring channels; the lanes of a head are neighbours in a warp, which sums the norm and swaps
// the halves of a rotation through shuffles.  A thread takes several sequences: the convolution's weights
// are read once (taps first, so that lanes read neighbouring bytes), and the next sequence's inputs are on
// their way while this one is worked on.  All slots of a ring are read in their own order, without waiting
// for the position, which only says which weight each meets.  Between the steps values stay in fp32;
// q, k and v are rounded once.
//
// Measured (device time): 1024 x 6144 bf16 with K = 4, RMS and rotation in 24.4 us, 3.1 TB/s (0.48 of the measured copy
// rate), fp32 without the rotation in 27.4 us; 1 x 2304 in 2.2 us, an empty launch.  Bound by latency at 500 threads an
// SM: with 80 or 64 registers a thread there are more, but they spill (35 and 53 us).
#include <algorithm>

#include "attn_common.cuh"
#include "host_util.h"
#include "kata_b200.h"

namespace kata {
namespace {

struct StepParams {
  const void* x;
  const long long* pos;
  void* ring;
  void* q;
  void* k;
  void* v;
  const float* conv_w;
  const float* qw;
  const float* kw;
  const float* cos;
  const float* sin;
  long long ldx;
  int B, HQ, H, D, Dv, norm_q, norm_k, rope, R, T;
  float eps_q, eps_k;
  int lph;   // lanes per head slot, a power of two
  int rows;  // sequences per thread
};

constexpr int kQT = 128;

// Eight neighbours as they lie in memory
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32<T>(reinterpret_cast<const T*>(w)[i]); }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <typename T, int K>
__global__ void __launch_bounds__(kQT) qkv_step_kernel(const StepParams p) {
  const int slots = p.HQ + 2 * p.H;
  const int spc = kQT / p.lph;  // head slots per CTA
  const int slot = blockIdx.x * spc + threadIdx.x / p.lph;
  const int e0 = (threadIdx.x % p.lph) * 8, lane = threadIdx.x & 31;
  const int kind = slot < p.HQ ? 0 : slot < p.HQ + p.H ? 1 : 2;
  const int dim = kind == 2 ? p.Dv : p.D;
  const bool live = slot < slots && e0 < dim;
  const int C = (p.HQ + p.H) * p.D + p.H * p.Dv;
  const int head = kind == 0 ? slot : kind == 1 ? slot - p.HQ : slot - p.HQ - p.H;
  const int c0 = (kind == 0 ? 0 : kind == 1 ? p.HQ * p.D : (p.HQ + p.H) * p.D) + head * dim + e0;
  const int norm = kind == 0 ? p.norm_q : kind == 1 ? p.norm_k : 0;
  const float* nw = kind == 0 ? p.qw : kind == 1 ? p.kw : nullptr;
  const float eps = kind == 0 ? p.eps_q : p.eps_k;

  float w[K ? K : 1][8];
  if (K && live) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const float4 lo = __ldg(reinterpret_cast<const float4*>(p.conv_w + static_cast<size_t>(j) * C + c0));
      const float4 hi = __ldg(reinterpret_cast<const float4*>(p.conv_w + static_cast<size_t>(j) * C + c0) + 1);
      w[j][0] = lo.x, w[j][1] = lo.y, w[j][2] = lo.z, w[j][3] = lo.w;
      w[j][4] = hi.x, w[j][5] = hi.y, w[j][6] = hi.z, w[j][7] = hi.w;
    }
  }
  constexpr int S = K > 1 ? K - 1 : 0;  // slots of a ring
  const int b_lo = blockIdx.y * p.rows, b_hi = min(b_lo + p.rows, p.B);
  Eight<T> nx, no[S ? S : 1];  // the next sequence's input and ring
  long long npos = 0;
  auto fetch = [&](int b) {
    npos = p.pos[b];
    if (!live) return;
    nx.load(static_cast<const T*>(p.x) + b * p.ldx + c0);
#pragma unroll
    for (int j = 0; j < S; ++j) no[j].load(static_cast<const T*>(p.ring) + (static_cast<size_t>(b) * S + j) * C + c0);
  };
  fetch(b_lo);
  for (int b = b_lo; b < b_hi; ++b) {
    const long long pos = npos;
    const Eight<T> xin = nx;
    Eight<T> old[S ? S : 1];
#pragma unroll
    for (int j = 0; j < S; ++j) old[j] = no[j];
    if (b + 1 < b_hi) fetch(b + 1);
    const bool bad = pos < 0 || (p.rope && pos >= p.T);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = live ? xin[i] : 0.f;
    if (K > 0 && live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= w[K ? K - 1 : 0][i];
      if constexpr (S > 0) {
        const int at = bad ? 0 : static_cast<int>(static_cast<unsigned long long>(pos) % S);
        // input pos - S + j is in slot (pos + j) % S: slot s meets weight (s - at) mod S
#pragma unroll
        for (int s = 0; s < S; ++s) {
          int j = s - at;
          if (j < 0) j += S;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float wj = w[0][i];
#pragma unroll
            for (int t = 1; t < S; ++t) wj = j == t ? w[t][i] : wj;
            y[i] = fmaf(wj, old[s][i], y[i]);
          }
        }
        if (!bad) xin.store(static_cast<T*>(p.ring) + (static_cast<size_t>(b) * S + at) * C + c0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4)
          y[i] = y[i] / (1.f + expf(-y[i]));
        else  // some ten units of fp32 at |a| near 10, far below the 2^-11 and 2^-8 of the outputs
          y[i] = __fdividef(y[i], 1.f + __expf(-y[i]));
      }
    }
    if (p.norm_q | p.norm_k) {  // the same for the whole warp, whose heads may be of all three kinds
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
      for (int o = p.lph / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float s = rsqrtf((norm == 2 ? ss / dim : ss) + eps);
      if (norm && live) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= (norm == 2 && nw) ? s * nw[e0 + i] : s;
      }
    }
    if (p.rope == 1 && kind < 2 && live) {
      const size_t at = static_cast<size_t>(bad ? 0 : pos) * (p.R / 2) + e0 / 2;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float c = p.cos[at + i / 2], s = p.sin[at + i / 2], a0 = y[i], a1 = y[i + 1];
        y[i] = a0 * c - a1 * s;
        y[i + 1] = a0 * s + a1 * c;
      }
    } else if (p.rope == 2) {
      const int half = p.R / 2, r0 = e0 % p.R;
      const bool first = r0 < half;
      float o[8];
      const int from = first ? lane + half / 8 : lane - half / 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, y[i], from & 31);
      if (kind < 2 && live) {
        const size_t at = static_cast<size_t>(bad ? 0 : pos) * half + (first ? r0 : r0 - half);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = p.cos[at + i], s = p.sin[at + i];
          y[i] = first ? y[i] * c - o[i] * s : y[i] * c + o[i] * s;
        }
      }
    }
    if (live) {
      if (bad) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7fffffff);
      }
      T* out = kind == 0 ? static_cast<T*>(p.q) + (static_cast<size_t>(b) * p.HQ + head) * p.D
               : kind == 1 ? static_cast<T*>(p.k) + (static_cast<size_t>(b) * p.H + head) * p.D
                           : static_cast<T*>(p.v) + (static_cast<size_t>(b) * p.H + head) * p.Dv;
      store8<T>(out + e0, y);
    }
  }
}

template <typename T>
void launch_step(const StepParams& p, int K, cudaStream_t st) {
  const int spc = kQT / p.lph, slots = p.HQ + 2 * p.H;
  const dim3 grid((slots + spc - 1) / spc, (p.B + p.rows - 1) / p.rows);
  switch (K) {
    case 0: qkv_step_kernel<T, 0><<<grid, kQT, 0, st>>>(p); break;
    case 1: qkv_step_kernel<T, 1><<<grid, kQT, 0, st>>>(p); break;
    case 2: qkv_step_kernel<T, 2><<<grid, kQT, 0, st>>>(p); break;
    case 3: qkv_step_kernel<T, 3><<<grid, kQT, 0, st>>>(p); break;
    default: qkv_step_kernel<T, 4><<<grid, kQT, 0, st>>>(p); break;
  }
}

}  // namespace
}  // namespace kata

using namespace kata;

extern "C" int kata_qkv_step(const kata_qkv_step_args* a, const void* x, long long ldx, const int64_t* positions,
                             void* ring, void* q, void* k, void* v, long long B, kata_stream_t stream) {
  if (!a) return KATA_ERR_INVALID;
  if (a->dtype != KATA_DTYPE_F32 && a->dtype != KATA_DTYPE_BF16 && a->dtype != KATA_DTYPE_F16) return KATA_ERR_DTYPE;
  if (B < 0 || B > 0x7fffffff || a->H < 1 || a->HQ < a->H || a->HQ % a->H || a->HQ > 65536) return KATA_ERR_SHAPE;
  if (a->D < 8 || a->D > 256 || a->D % 8 || a->Dv < 8 || a->Dv > 256 || a->Dv % 8) return KATA_ERR_SHAPE;
  if (a->K < 0 || a->K > 4) return KATA_ERR_UNSUPPORTED;
  if (a->norm_q < 0 || a->norm_q > 2 || a->norm_k < 0 || a->norm_k > 2 || a->rope < 0 || a->rope > 2) return KATA_ERR_INVALID;
  if (a->rope) {
    if (!a->cos || !a->sin || a->T < 1) return KATA_ERR_INVALID;
    if (a->rope == 1 && a->R != a->D) return KATA_ERR_SHAPE;
    if (a->rope == 2 && (a->R < 16 || a->R % 16 || a->D % a->R)) return KATA_ERR_SHAPE;
  }
  if (a->K > 0 && !a->conv_w) return KATA_ERR_INVALID;
  const int C = (a->HQ + a->H) * a->D + a->H * a->Dv;
  if (B > 1 && ldx < C) return KATA_ERR_SHAPE;
  if (B == 0) return KATA_OK;
  if (!x || !positions || !q || !k || !v || (a->K > 1 && !ring)) return KATA_ERR_INVALID;
  auto al = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; };
  if (!al(a->conv_w) || !al(x) || !al(q) || !al(k) || !al(v) || (a->K > 1 && !al(ring)) || ldx % (a->dtype == KATA_DTYPE_F32 ? 4 : 8))
    return KATA_ERR_ALIGN;
  StepParams p;
  p.x = x;
  p.pos = reinterpret_cast<const long long*>(positions);
  p.ring = ring;
  p.q = q;
  p.k = k;
  p.v = v;
  p.conv_w = a->conv_w;
  p.qw = a->q_weight;
  p.kw = a->k_weight;
  p.cos = a->cos;
  p.sin = a->sin;
  p.ldx = ldx;
  p.B = static_cast<int>(B);
  p.HQ = a->HQ;
  p.H = a->H;
  p.D = a->D;
  p.Dv = a->Dv;
  p.norm_q = a->norm_q;
  p.norm_k = a->norm_k;
  p.rope = a->rope;
  p.R = a->R;
  p.T = a->T;
  p.eps_q = a->eps_q;
  p.eps_k = a->eps_k;
  int lph = 1;
  while (lph * 8 < std::max(a->D, a->Dv)) lph *= 2;
  p.lph = lph;
  // several sequences a thread once the grid fills the GPU several times over (1024 x 6144: 31.3 us with one, 25.6
  // with three or more)
  const long long ctas = ((a->HQ + 2ll * a->H) * lph + kQT - 1) / kQT * B;
  p.rows = static_cast<int>(std::max<long long>(std::min<long long>(4, ctas / (148 * 8)), (B + 65534) / 65535));
  p.rows = std::max(p.rows, 1);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == KATA_DTYPE_BF16)
    launch_step<__nv_bfloat16>(p, a->K, st);
  else if (a->dtype == KATA_DTYPE_F16)
    launch_step<__half>(p, a->K, st);
  else
    launch_step<float>(p, a->K, st);
  return from_cuda(cudaGetLastError());
}
