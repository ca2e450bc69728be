// w4.cu -- linear layer with 4-bit weights and group scales: y = x W^T,
//   W[n,k] = scale[n, k/g] (code[n,k] - zero[n, k/g]),  y[m,n] = sum_G scale[n,G] sum_{k in G} (code - zero) x[m,k].
//
// Layout (written once by kata_w4_pack).  Rows go in tiles of 16, k in steps of 128; a tile's steps and
// the tiles themselves are contiguous, so that a run of work is one run of memory.  A step of a tile is
// 1 KB: [row half][lane][block of 32 k] words of 8 codes, lane = 4 (row % 8) + q holding codes 8q..8q+7
// of each block, which are exactly the lane's A-fragment values of mma.m16n8k16 (two MMAs a block, the
// k slots of an MMA being codes 8q + 4j + {0,1} and {2,3} of the four lanes q).  Nibble i of a word is
// code 2i and nibble i + 4 code 2i + 1, so that (word >> 4i) & 0x000f000f is a pair of neighbours.
// Scales (and zeros) follow as [tile][group][16 rows].  A gated weight's tile holds 8 gate rows and the
// 8 up rows that belong to them, so that both sums of an output end in the same lane.
#include <algorithm>

#include "attn_common.cuh"
#include "host_util.h"
#include "sm100.cuh"

namespace kata {
namespace {

constexpr int kStepBytes = 1024;  // codes of 16 rows x 128 k

struct W4Geom {
  int tiles, steps;  // row tiles, steps of 128 k
  int gps;           // groups a step spans (4, 2 or 1)
  int spg;           // steps a group spans (1 unless group > 128)
  int groups;        // groups stored per tile: every step's run is whole
};

inline W4Geom w4_geom(const kata_w4_weight* w) {
  W4Geom g;
  g.tiles = w->gated ? (w->N / 2 + 7) / 8 : (w->N + 15) / 16;
  g.steps = (w->K + 127) / 128;
  g.gps = w->group < 128 ? 128 / w->group : 1;
  g.spg = w->group > 128 ? w->group / 128 : 1;
  g.groups = w->group <= 128 ? g.steps * g.gps : (g.steps + g.spg - 1) / g.spg;
  return g;
}

// The weight row that row r (0..15) of tile t holds, or -1 for padding.
__host__ __device__ inline int w4_row(int t, int r, int N, int gated) {
  if (!gated) {
    const int n = t * 16 + r;
    return n < N ? n : -1;
  }
  const int n = t * 8 + (r & 7);
  return n < N / 2 ? n + (r >> 3) * (N / 2) : -1;
}

// One thread per word of the laid-out codes; then the scales and zeros of each (tile, group, row).
__global__ void __launch_bounds__(256) w4_pack_codes_kernel(const uint32_t* __restrict__ packed,
                                                            uint32_t* __restrict__ codes, int N, int K, int gated,
                                                            int steps, long long words) {
  const int wpr = 4 * ((K + 31) / 32);  // words a row of the input has
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < words; i += gridDim.x * 256ll) {
    const int b = i & 3, lane = (i >> 2) & 31, half = (i >> 7) & 1;
    const long long f = i >> 8;
    const int step = static_cast<int>(f % steps), t = static_cast<int>(f / steps);
    const int n = w4_row(t, half * 8 + (lane >> 2), N, gated);
    const int src = step * 16 + b * 4 + (lane & 3);
    uint32_t v = 0x88888888u;
    if (n >= 0 && src < wpr) v = packed[static_cast<size_t>(n) * wpr + src];
    uint32_t o = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o |= ((v >> (8 * j)) & 15u) << (4 * j);
      o |= ((v >> (8 * j + 4)) & 15u) << (4 * j + 16);
    }
    codes[i] = o;
  }
}

template <typename S>
__global__ void __launch_bounds__(256) w4_pack_scales_kernel(const S* __restrict__ scales, S* __restrict__ out, int N,
                                                             int G, int gated, int groups, long long n_out, S fill) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n_out; i += gridDim.x * 256ll) {
    const long long f = i >> 4;
    const int g = static_cast<int>(f % groups), t = static_cast<int>(f / groups);
    const int n = w4_row(t, static_cast<int>(i & 15), N, gated);
    out[i] = (n >= 0 && g < G) ? scales[static_cast<size_t>(n) * G + g] : fill;
  }
}

// ------------------------------------------------------------------------------------------------
// Streaming kernel: few rows of x, the codes read once from HBM.
// ------------------------------------------------------------------------------------------------

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes to 16-bit floats: a nibble ORed into the mantissa of 128 (bf16) or 1024 (f16) is 128 + code or
// 1024 + code exactly; from there one fused multiply-add leaves unit (code - zero) exactly.  With bf16
// the unit is 2^-10: a group's sum of unscaled products stays finite for every finite x.  f16 values are
// too small to come near the end of fp32 (unit 1).  The scale takes the unit back.
template <typename T>
struct Magic;
template <>
struct Magic<__nv_bfloat16> {
  static constexpr uint32_t base = 0x43004300u;   // 128
  static constexpr uint32_t unit = 0x3a803a80u;   // 2^-10
  static constexpr float back = 1024.f;
  // -(128 + zero) 2^-10
  static __device__ __forceinline__ uint32_t offset(uint32_t zero) {
    const __nv_bfloat162 v = __float2bfloat162_rn(-(128.f + static_cast<float>(zero)) * (1.f / 1024.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b) {
    const uint32_t u = unit;
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&u),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Magic<__half> {
  static constexpr uint32_t base = 0x64006400u;   // 1024
  static constexpr float back = 1.f;
  // -(1024 + zero)
  static __device__ __forceinline__ uint32_t offset(uint32_t zero) { return 0xe400e400u + 0x00010001u * zero; }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b) {
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <typename T>
__device__ __forceinline__ uint32_t dequant_pair(uint32_t word, int i, uint32_t offset) {
  return Magic<T>::fma2(((word >> (4 * i)) & 0x000f000fu) | Magic<T>::base, offset);
}

// An fp32 value as three bf16 parts, each the leading 8 bits of what is left: exact together, and no
// part overflows.  Infinities and NaN stay in the first part.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  const float a = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const bool fin = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
  const float r = fin ? x - a : 0.f;
  const float b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  p[0] = __float2bfloat16_rn(fin ? a : x);
  p[1] = __float2bfloat16_rn(b);
  p[2] = __float2bfloat16_rn(r - b);
}

struct W4Params {
  const unsigned char* codes;
  const unsigned char* scales;
  const unsigned char* zeros;
  const void* x;
  void* y;
  long long ldx, ldy;
  int rows, N, K, gated;
  W4Geom g;
  int tpb;          // row tiles a CTA works on at once (its partial sums are kept in shared memory)
  int chunk_steps;  // steps of k whose x is in shared memory at once
  int stage_bytes;
};

constexpr int kWarps = 8;
constexpr int kDepth = 6;  // steps in flight per warp

// T: operand type of the products; X: type of x, y and the scales (float: PARTS = 3 columns a row).
// NT: tiles of 8 columns.  GPS: groups per step.
template <typename T, typename X, int NT, int GPS, bool ZERO>
__global__ void __launch_bounds__(kWarps * 32) w4_stream_kernel(const W4Params p) {
  constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
  constexpr int COLS = 8 * NT;
  constexpr int ROWS = COLS / PARTS;  // rows of x a CTA takes
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = blockIdx.y * ROWS;
  const int nrow = min(ROWS, p.rows - row0), ncol = nrow * PARTS;
  const int kc = p.chunk_steps * 128;
  const int pitch = kc + 32;  // 64 bytes more than a multiple of 256: the eight 16-byte reads of a quarter warp
                              // (two columns, four q) fall on all 32 banks
  T* xs = reinterpret_cast<T*>(smem);
  unsigned char* ring = smem + static_cast<size_t>(min(COLS, p.rows * PARTS)) * pitch * sizeof(T);
  float* red = reinterpret_cast<float*>(ring + kWarps * kDepth * p.stage_bytes);
  unsigned char* myring = ring + warp * kDepth * p.stage_bytes;
  const uint32_t myring_s = smem_u32(myring);

  // this CTA's tiles, as even as whole tiles allow
  const int t_lo = static_cast<int>(static_cast<long long>(p.g.tiles) * blockIdx.x / gridDim.x);
  const int t_hi = static_cast<int>(static_cast<long long>(p.g.tiles) * (blockIdx.x + 1) / gridDim.x);
  const int g = lane >> 2, q = lane & 3;
  const int chunks = (p.g.steps + p.chunk_steps - 1) / p.chunk_steps;
  const X* x = static_cast<const X*>(p.x) + row0 * p.ldx;
  const int bcol = min(g, ncol - 1);  // columns past the last hold what nobody reads

  for (int tb = t_lo; tb < t_hi; tb += p.tpb) {
    const int nt = min(p.tpb, t_hi - tb);
    const int total = nt * p.chunk_steps;
    const int f_lo = total * warp / kWarps, f_hi = total * (warp + 1) / kWarps;
    for (int ch = 0; ch < chunks; ++ch) {
      const int s0 = ch * p.chunk_steps;
      const int ns = min(p.chunk_steps, p.g.steps - s0);
      if (ch > 0 || (tb > t_lo && chunks > 1)) __syncthreads();  // the chunk before is no longer read
      if (tb == t_lo || chunks > 1) {
        const int k0 = s0 * 128;
        const bool vec = sizeof(X) == 2 && (p.ldx % 8) == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0;
        for (int i = tid; i < nrow * (kc / 8); i += kWarps * 32) {
          const int r = i / (kc / 8), k = (i - r * (kc / 8)) * 8;
          const X* src = x + r * p.ldx + k0 + k;
          if (vec && k0 + k + 8 <= p.K) {
            *reinterpret_cast<uint4*>(xs + r * pitch + k) = *reinterpret_cast<const uint4*>(src);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const X v = k0 + k + j < p.K ? src[j] : from_f32<X>(0.f);
              if constexpr (PARTS == 1) {
                xs[r * pitch + k + j] = v;
              } else {
                __nv_bfloat16 s3[3];
                split3(v, s3);
#pragma unroll
                for (int c = 0; c < 3; ++c) xs[(r * 3 + c) * pitch + k + j] = s3[c];
              }
            }
          }
        }
        __syncthreads();
      }

      // this warp's run of (tile, step); `it`, `is` are where the next copy goes
      int it = f_lo / p.chunk_steps, is = f_lo - it * p.chunk_steps;
      int ct = it, cs = is;
      int fi = f_lo;
      auto issue = [&]() {
        if (fi < f_hi && is < ns) {
          const uint32_t dst = myring_s + ((fi - f_lo) % kDepth) * p.stage_bytes;
          const long long f = static_cast<long long>(tb + it) * p.g.steps + s0 + is;
          const unsigned char* src = p.codes + f * kStepBytes;
          cp_async16(dst + lane * 16, src + lane * 16);
          cp_async16(dst + 512 + lane * 16, src + 512 + lane * 16);
          const long long gi = p.g.spg == 1 ? f * GPS : static_cast<long long>(tb + it) * p.g.groups + (s0 + is) / p.g.spg;
          constexpr int SB = GPS * 16 * static_cast<int>(sizeof(X));  // scales of a step
#pragma unroll
          for (int o = 0; o < SB; o += 128)
            if (o + lane * 4 < SB) cp_async4(dst + kStepBytes + o + lane * 4, p.scales + gi * 16 * sizeof(X) + o + lane * 4);
          if (ZERO && lane < GPS * 4) cp_async4(dst + kStepBytes + SB + lane * 4, p.zeros + gi * 16 + lane * 4);
        }
        cp_async_commit();
        ++fi;
        if (++is == p.chunk_steps) {
          is = 0;
          ++it;
        }
      };
#pragma unroll
      for (int d = 0; d < kDepth - 1; ++d) issue();

      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
      for (int f = f_lo; f < f_hi; ++f) {
        cp_async_wait<kDepth - 2>();
        __syncwarp();  // every lane's copies of this step are in, and the step before is no longer read
        issue();
        if (cs < ns) {
          const unsigned char* st = myring + ((f - f_lo) % kDepth) * p.stage_bytes;
          const uint4 w0 = *reinterpret_cast<const uint4*>(st + lane * 16);
          const uint4 w1 = *reinterpret_cast<const uint4*>(st + 512 + lane * 16);
          const uint32_t wa[4] = {w0.x, w0.y, w0.z, w0.w}, wb[4] = {w1.x, w1.y, w1.z, w1.w};
          const X* sc = reinterpret_cast<const X*>(st + kStepBytes);
          const unsigned char* zp = st + kStepBytes + GPS * 16 * sizeof(X);
          float part[NT][4];
          uint32_t z0 = Magic<T>::offset(8), z1 = z0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (b % (4 / GPS) == 0) {
#pragma unroll
              for (int n = 0; n < NT; ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f;
              if (ZERO) {
                z0 = Magic<T>::offset(zp[(b * GPS / 4) * 16 + g] & 15u);
                z1 = Magic<T>::offset(zp[(b * GPS / 4) * 16 + g + 8] & 15u);
              }
            }
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              a[j][0] = dequant_pair<T>(wa[b], 2 * j, z0);
              a[j][1] = dequant_pair<T>(wb[b], 2 * j, z1);
              a[j][2] = dequant_pair<T>(wa[b], 2 * j + 1, z0);
              a[j][3] = dequant_pair<T>(wb[b], 2 * j + 1, z1);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int col = NT == 1 ? bcol : min(n * 8 + g, ncol - 1);
              const uint4 xv = *reinterpret_cast<const uint4*>(xs + col * pitch + cs * 128 + b * 32 + q * 8);
              mma16816(part[n], a[0], xv.x, xv.y, T());
              mma16816(part[n], a[1], xv.z, xv.w, T());
            }
            if (b % (4 / GPS) == 4 / GPS - 1) {
              const float s0f = to_f32<X>(sc[(b * GPS / 4) * 16 + g]) * Magic<T>::back;
              const float s1f = to_f32<X>(sc[(b * GPS / 4) * 16 + g + 8]) * Magic<T>::back;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                acc[n][0] = fmaf(s0f, part[n][0], acc[n][0]);
                acc[n][1] = fmaf(s0f, part[n][1], acc[n][1]);
                acc[n][2] = fmaf(s1f, part[n][2], acc[n][2]);
                acc[n][3] = fmaf(s1f, part[n][3], acc[n][3]);
              }
            }
          }
        }
        if (++cs == p.chunk_steps || f + 1 == f_hi) {
          // the tile's part of this warp: tiles and warps grow together along the run, so tile + warp
          // is a slot of its own
          float* slot = red + static_cast<size_t>(ct + warp) * 16 * COLS;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float* d = slot + (g + (e >> 1) * 8) * COLS + n * 8 + 2 * q + (e & 1);
              *d = ch == 0 ? acc[n][e] : *d + acc[n][e];
              acc[n][e] = 0.f;
            }
          }
          if (cs == p.chunk_steps) {
            cs = 0;
            ++ct;
          }
        }
      }
      cp_async_wait<0>();
    }
    __syncthreads();
    // Sums over the warps that had a part of the tile, in warp order.
    const int orow = p.gated ? 8 : 16;
    for (int i = tid; i < nt * orow * nrow; i += kWarps * 32) {
      const int r = i % orow, rest = i / orow;
      const int m = rest % nrow, t = rest / nrow;
      float s = 0.f, s2 = 0.f;
      for (int w = 0; w < kWarps; ++w) {
        const int a = total * w / kWarps, b = total * (w + 1) / kWarps;
        if (a >= b || a >= (t + 1) * p.chunk_steps || b <= t * p.chunk_steps) continue;
        const float* slot = red + static_cast<size_t>(t + w) * 16 * COLS;
#pragma unroll
        for (int c = 0; c < PARTS; ++c) {
          s += slot[r * COLS + m * PARTS + c];
          if (p.gated) s2 += slot[(r + 8) * COLS + m * PARTS + c];
        }
      }
      const int n = (tb + t) * orow + r;
      if (n < (p.gated ? p.N / 2 : p.N)) {
        if (p.gated) s = s / (1.f + expf(-s)) * s2;
        static_cast<X*>(p.y)[(row0 + m) * p.ldy + n] = from_f32<X>(s);
      }
    }
    __syncthreads();
  }
}

template <typename T, typename X, int NT, int GPS, bool ZERO>
int launch_stream(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows,
                  cudaStream_t st) {
  constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
  constexpr int COLS = 8 * NT;
  W4Params p;
  p.codes = static_cast<const unsigned char*>(w->codes);
  p.scales = static_cast<const unsigned char*>(w->scales);
  p.zeros = static_cast<const unsigned char*>(w->zeros);
  p.x = x;
  p.y = y;
  p.ldx = ldx;
  p.ldy = ldy;
  p.rows = rows;
  p.N = w->N;
  p.K = w->K;
  p.gated = w->gated;
  p.g = w4_geom(w);
  p.stage_bytes = kStepBytes + GPS * 16 * static_cast<int>(sizeof(X)) + (ZERO ? GPS * 16 : 0);
  const int ccols = std::min(COLS, rows * PARTS);
  const int slabs = (rows * PARTS + COLS / PARTS * PARTS - 1) / (COLS / PARTS * PARTS);
  // x of as many steps as fit 96 KB, in chunks of one length
  const int fit = std::max(1, (96 * 1024 / (ccols * 2) - 32) / 128);
  const int chunks = (p.g.steps + fit - 1) / fit;
  p.chunk_steps = (p.g.steps + chunks - 1) / chunks;
  const int grid = std::min(p.g.tiles, std::max(1, 148 * 2 / slabs));
  p.tpb = std::min(8, (p.g.tiles + grid - 1) / grid);
  const size_t smem = static_cast<size_t>(ccols) * (p.chunk_steps * 128 + 32) * 2 + kWarps * kDepth * p.stage_bytes +
                      static_cast<size_t>(p.tpb + kWarps - 1) * 16 * COLS * 4;
  auto kern = w4_stream_kernel<T, X, NT, GPS, ZERO>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return KATA_ERR_CUDA;
  kern<<<dim3(grid, slabs), kWarps * 32, smem, st>>>(p);
  return from_cuda(cudaGetLastError());
}

template <typename T, typename X, int NT>
int launch_groups(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows,
                  cudaStream_t st) {
  const int gps = w->group < 128 ? 128 / w->group : 1;
  if (w->zeros) {
    if (gps == 4) return launch_stream<T, X, NT, 4, true>(w, x, ldx, y, ldy, rows, st);
    if (gps == 2) return launch_stream<T, X, NT, 2, true>(w, x, ldx, y, ldy, rows, st);
    return launch_stream<T, X, NT, 1, true>(w, x, ldx, y, ldy, rows, st);
  }
  if (gps == 4) return launch_stream<T, X, NT, 4, false>(w, x, ldx, y, ldy, rows, st);
  if (gps == 2) return launch_stream<T, X, NT, 2, false>(w, x, ldx, y, ldy, rows, st);
  return launch_stream<T, X, NT, 1, false>(w, x, ldx, y, ldy, rows, st);
}

template <typename T, typename X>
int launch_rows(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows,
                cudaStream_t st) {
  const int cols = rows * (sizeof(X) == 4 ? 3 : 1);
  if (cols <= (sizeof(X) == 4 ? 6 : 8)) return launch_groups<T, X, 1>(w, x, ldx, y, ldy, rows, st);
  if (cols <= (sizeof(X) == 4 ? 15 : 16)) return launch_groups<T, X, 2>(w, x, ldx, y, ldy, rows, st);
  return launch_groups<T, X, 4>(w, x, ldx, y, ldy, rows, st);
}

int w4_check(const kata_w4_weight* w) {
  if (!w) return KATA_ERR_INVALID;
  if (w->dtype != KATA_DTYPE_F32 && w->dtype != KATA_DTYPE_BF16 && w->dtype != KATA_DTYPE_F16) return KATA_ERR_DTYPE;
  if (w->N < 1 || w->K < 1 || w->N > (1 << 24) || w->K > (1 << 24)) return KATA_ERR_SHAPE;
  if (w->group != 32 && w->group != 64 && (w->group < 128 || w->group % 128)) return KATA_ERR_SHAPE;
  if (w->gated != 0 && w->gated != 1) return KATA_ERR_INVALID;
  if (w->gated && w->N % 2) return KATA_ERR_SHAPE;
  return KATA_OK;
}

size_t w4_esize(int dtype) { return dtype == KATA_DTYPE_F32 ? 4 : 2; }
bool w4_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kata

using namespace kata;

extern "C" int kata_w4_layout(const kata_w4_weight* w, size_t* code_bytes, size_t* scale_bytes, size_t* zero_bytes) {
  if (int e = w4_check(w)) return e;
  const W4Geom g = w4_geom(w);
  if (code_bytes) *code_bytes = static_cast<size_t>(g.tiles) * g.steps * kStepBytes;
  if (scale_bytes) *scale_bytes = static_cast<size_t>(g.tiles) * g.groups * 16 * w4_esize(w->dtype);
  if (zero_bytes) *zero_bytes = static_cast<size_t>(g.tiles) * g.groups * 16;
  return KATA_OK;
}

extern "C" int kata_w4_pack(const void* packed, const void* scales, const void* zeros, const kata_w4_weight* w,
                            kata_stream_t stream) {
  if (int e = w4_check(w)) return e;
  if (!packed || !scales || !w->codes || !w->scales || (!zeros) != (!w->zeros)) return KATA_ERR_INVALID;
  if (!w4_al16(w->codes) || !w4_al16(w->scales) || (w->zeros && !w4_al16(w->zeros))) return KATA_ERR_ALIGN;
  const W4Geom g = w4_geom(w);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long words = static_cast<long long>(g.tiles) * g.steps * (kStepBytes / 4);
  const long long ns = static_cast<long long>(g.tiles) * g.groups * 16;
  const int G = (w->K + w->group - 1) / w->group;
  auto grid = [](long long n) { return static_cast<int>(std::min<long long>(148 * 16, (n + 255) / 256)); };
  w4_pack_codes_kernel<<<grid(words), 256, 0, st>>>(static_cast<const uint32_t*>(packed),
                                                    static_cast<uint32_t*>(const_cast<void*>(w->codes)), w->N, w->K,
                                                    w->gated, g.steps, words);
  if (w->dtype == KATA_DTYPE_F32)
    w4_pack_scales_kernel<uint32_t><<<grid(ns), 256, 0, st>>>(static_cast<const uint32_t*>(scales),
                                                              static_cast<uint32_t*>(const_cast<void*>(w->scales)), w->N,
                                                              G, w->gated, g.groups, ns, 0u);
  else
    w4_pack_scales_kernel<uint16_t><<<grid(ns), 256, 0, st>>>(static_cast<const uint16_t*>(scales),
                                                              static_cast<uint16_t*>(const_cast<void*>(w->scales)), w->N,
                                                              G, w->gated, g.groups, ns, static_cast<uint16_t>(0));
  if (zeros)
    w4_pack_scales_kernel<uint8_t><<<grid(ns), 256, 0, st>>>(static_cast<const uint8_t*>(zeros),
                                                             static_cast<uint8_t*>(const_cast<void*>(w->zeros)), w->N, G,
                                                             w->gated, g.groups, ns, static_cast<uint8_t>(8));
  return from_cuda(cudaGetLastError());
}

extern "C" int kata_w4_linear(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy,
                              long long rows, int* status, kata_stream_t stream) {
  if (int e = w4_check(w)) return e;
  if (rows < 0 || rows > (1ll << 30)) return KATA_ERR_SHAPE;
  if (rows == 0) return KATA_OK;
  if (!w->codes || !w->scales || !x || !y) return KATA_ERR_INVALID;
  if (!w4_al16(w->codes) || !w4_al16(w->scales) || (w->zeros && !w4_al16(w->zeros))) return KATA_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(x) % w4_esize(w->dtype) || reinterpret_cast<uintptr_t>(y) % w4_esize(w->dtype))
    return KATA_ERR_ALIGN;
  if (rows > 1 && (ldx < w->K || ldy < (w->gated ? w->N / 2 : w->N))) return KATA_ERR_SHAPE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int slab = w->dtype == KATA_DTYPE_F32 ? 10 : 32;  // rows per slab of the widest form; slabs are the grid's y
  for (long long r = 0; r < rows; r += 65535ll * slab) {
    const int n = static_cast<int>(std::min<long long>(rows - r, 65535ll * slab));
    const unsigned char* xr = static_cast<const unsigned char*>(x) + r * ldx * w4_esize(w->dtype);
    unsigned char* yr = static_cast<unsigned char*>(y) + r * ldy * w4_esize(w->dtype);
    int e;
    if (w->dtype == KATA_DTYPE_BF16)
      e = launch_rows<__nv_bfloat16, __nv_bfloat16>(w, xr, ldx, yr, ldy, n, st);
    else if (w->dtype == KATA_DTYPE_F16)
      e = launch_rows<__half, __half>(w, xr, ldx, yr, ldy, n, st);
    else
      e = launch_rows<__nv_bfloat16, float>(w, xr, ldx, yr, ldy, n, st);
    if (e) return e;
  }
  (void)status;
  return KATA_OK;
}
