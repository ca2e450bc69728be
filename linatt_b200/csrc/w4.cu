// w4.cu -- linear layer with 4-bit weights and group scales: y = x W^T,
//   W[n,k] = scale[n, k/g] (code[n,k] - zero[n, k/g]),  y[m,n] = sum_G scale[n,G] sum_{k in G} (code - zero) x[m,k].
//
// Layout (written once by kata_w4_pack).  Rows go in tiles of 16, k in steps of 128; a tile's steps and
// the tiles themselves are contiguous, so that a run of work is one run of memory.  A step of a tile is
// 1 KB: [row half][lane][block of 32 k] words of 8 codes, lane = 4 (row % 8) + q holding codes 8q..8q+7
// of each block: byte j of a word has code j in its low and code j + 4 in its high nibble, so that
// word & 0x0f0f0f0f and (word >> 4) & 0x0f0f0f0f are four neighbours as bytes -- as they are, the lane's
// A-fragment registers of mma.m16n8k32 on bytes (k slots 4q..4q+3 and 16+4q.. being codes 8q.. and 8q+4..).
// The step's scales, [group][16 rows], and zeros follow in the same record (a group of several steps is
// stored in each of them), so that a run of steps is one bulk copy.  A gated weight's tile holds 8 gate rows and the 8 up rows that belong to them.
#include <algorithm>

#include "attn_common.cuh"
#include "host_util.h"
#include "sm100.cuh"

namespace kata {
namespace {

constexpr int kMaxSmem = 232448;  // dynamic shared memory a CTA may have
constexpr int kStepBytes = 1024;  // codes of 16 rows x 128 k

struct W4Geom {
  int tiles, steps;  // row tiles, steps of 128 k
  int gps;           // groups of a step (4, 2 or 1; a group of several steps is stored once for each)
  int side;          // bytes of a step's scales and zeros
  int rec;           // bytes of a step
};

inline W4Geom w4_geom(const kata_w4_weight* w) {
  W4Geom g;
  g.tiles = w->gated ? (w->N / 2 + 7) / 8 : (w->N + 15) / 16;
  g.steps = (w->K + 127) / 128;
  g.gps = w->group < 128 ? 128 / w->group : 1;
  g.side = g.gps * 16 * ((w->dtype == KATA_DTYPE_F32 ? 4 : 2) + (w->zeros ? 1 : 0));
  g.rec = kStepBytes + g.side;
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

// One warp per record: its codes, then its scales and zeros.
template <typename S>
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint32_t* __restrict__ packed, const S* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros, unsigned char* __restrict__ data,
                                                      int N, int K, int group, int gated, W4Geom g) {
  const int wpr = 4 * ((K + 31) / 32);  // words a row of the input has
  const int G = (K + group - 1) / group, lane = threadIdx.x & 31;
  const long long records = static_cast<long long>(g.tiles) * g.steps;
  for (long long f = blockIdx.x * 8ll + (threadIdx.x >> 5); f < records; f += gridDim.x * 8ll) {
    const int step = static_cast<int>(f % g.steps), t = static_cast<int>(f / g.steps);
    unsigned char* rec = data + f * g.rec;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int n = w4_row(t, half * 8 + (lane >> 2), N, gated);
      uint32_t o[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int src = step * 16 + b * 4 + (lane & 3);
        const uint32_t v = n >= 0 && src < wpr ? packed[static_cast<size_t>(n) * wpr + src] : 0x88888888u;
        o[b] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[b] |= ((v >> (4 * j)) & 15u) << (8 * j) | ((v >> (4 * j + 16)) & 15u) << (8 * j + 4);
      }
      reinterpret_cast<uint4*>(rec)[half * 32 + lane] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    for (int i = lane; i < g.gps * 16; i += 32) {
      const int n = w4_row(t, i & 15, N, gated), gr = min((step * 128 + (i >> 4) * (128 / g.gps)) / group, G);
      const bool live = n >= 0 && gr < G;
      reinterpret_cast<S*>(rec + kStepBytes)[i] = live ? scales[static_cast<size_t>(n) * G + gr] : S(0);
      if (zeros) rec[kStepBytes + g.gps * 16 * sizeof(S) + i] = live ? zeros[static_cast<size_t>(n) * G + gr] : 8;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Streaming kernel: few rows of x, the codes read once from HBM.
//
// Turning codes into 16-bit floats costs 11 instructions a word and bounds such a kernel at half the HBM
// rate (measured: 1 x 8192 x 32768 in 36 us against 21 us for the bytes).  Bytes cost 3.  So x becomes
// whole numbers: the 128 values of a row's step are scaled by a power of two and split into signed base-256
// digits, each a column of the product, whose sums over a group are exact in 32 bits.  A group's sum of
// (code - 8) times a digit is below 2^22, so it is accumulated on top of the bits of 1.5 2^23 and is a float
// as it stands; -8 sum(digits) is part of that start.
//
// Nothing of x is lost.  What the digits leave of a value far below the largest of its 128 is a float again,
// and so is all of an infinity or NaN, which has no digits.  Where x is staged these rests are kept by blocks of 32
// (as many as there is room for, the others are formed again from x) and the row's step is marked; the warp
// that works on it adds rest times weight in fp32.  The digits are as many as make that rare: 3 a row reach to 2^-23
// of the largest, so that of normally distributed steps one in 200 (bf16) or 30 (f16) has a rest, 5 of fp32 to
// 2^-38, one in 100 (4 would leave one in two of three), and a single column tile has room for more.  What
// rests cost (device time): 5 x 8192 x 8192 f16 23.2 us, bf16 21.2; with a value 10^4 times the others in every
// eighth step 31.3.  What the digits of fp32 cost over 4 that would round x: 2 x 8192 x 8192 18.3 us against 12.9.
//
// Measured (device time): 1 x 8192 x 32768 in 24.7 us, 5.6 TB/s of codes and scales, 0.87 of the measured copy
// rate, but 1 x 8192 x 8192 in 10.1 us, 0.53, where the start of the kernel counts; 1 x 4096 x 4096 in 5.6 us;
// 1 x 768 x 768 in 3.4 us, where an empty launch takes 2: bound there by launch, by code that is fetched cold and by
// the two trips to memory that follow one another.
// ------------------------------------------------------------------------------------------------

__device__ __forceinline__ void imma16832(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct W4Params {
  const unsigned char* data;
  const void* x;
  void* y;
  long long ldx, ldy;
  int* status;
  int rows, N, K, gated;
  W4Geom g;
  int tiles_q, tiles_r;  // tiles of a CTA, and how many CTAs have one more
  int chunks;
  int tpb;          // row tiles a CTA works on at once (their sums are kept in shared memory)
  int chunk_steps;  // steps of k whose x is in shared memory at once
  int keep;         // blocks of 32 k whose rests are too
  int align;        // rows of x start on 16-byte boundaries, or 8-byte ones, or others (2)
  int wpr;          // warps that a row of x is staged by
  uint32_t by_steps, by_rows, by_wpr;  // reciprocals of chunk_steps, rows and wpr
};

// n / d through the reciprocal r = ceil(2^32 / d), for n d < 2^32 (a division costs 100 cycles of a call's 3000)
inline uint32_t recip(uint32_t d) { return d == 1 ? 0 : static_cast<uint32_t>((0x100000000ull + d - 1) / d); }
__device__ __forceinline__ int div_by(int n, uint32_t r) { return r ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), r)) : n; }

constexpr int kWarps = 16;
// steps per copy, at most: fewer where the scales are many, so that the rings leave room for x
constexpr int unit_of(int side_bytes) { return side_bytes > 96 ? 2 : 4; }
constexpr int kDepth = 2;  // copies in flight per warp
constexpr int kMagicBits = 0x4b400000;  // 1.5 2^23
constexpr float kMagic = 12582912.f;

// |x| < 0.9961 2^(e - 126) is x = 2^(e - 126 - top) (h + 2^-low l) and a rest: h of H digits, at most 0.9961 2^top,
// which is 127 (1 + 2^8 + ..), l of L, at most 2^(low - 1).  A column tile takes one row of 6 digits (fp32), two of 4
// (16-bit types); two and more tiles take 5 (3) a row.
template <typename X, int NT>
struct Digits {
  static constexpr int H = sizeof(X) == 2 && NT == 1 ? 4 : 3;
  static constexpr int L = sizeof(X) == 2 ? 0 : NT == 1 ? 3 : 2;
  static constexpr int N = H + L;
  static constexpr int top = H == 4 ? 31 : 23;
  static constexpr int low = L == 3 ? 23 : L == 2 ? 15 : 0;
  static constexpr int bits = top + low;
  static constexpr int rows() { return 8 * NT / N; }  // of x that NT tiles take
};
template <typename X>
constexpr int kPrecision = sizeof(X) == 4 ? 24 : std::is_same<X, __half>::value ? 11 : 8;  // bits that a value has
constexpr uint32_t kRoundUp = 0x10200;  // added to the bits of a float: to the next power of two from 1.99213 on
constexpr int kMarkRows = 16;           // a step's marks, one a row: its blocks with a rest, and from bit 4 on their place
constexpr int kMaxRests = 1024;         // blocks whose rests are kept

// Eight neighbours of a row of x as they are in memory (zeros past its end)
template <typename X>
struct Raw8 {
  uint4 w[sizeof(X) / 2];
  // align: bytes that the rows' starts are multiples of, 16, 8 or less
  __device__ __forceinline__ void load(const X* src, int left, int align) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(X) / 2); ++i) w[i] = make_uint4(0, 0, 0, 0);
    if (align == 16 && left >= 8) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(X) / 2); ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    } else if (align == 8 && left >= 8) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(X)); ++i)
        reinterpret_cast<uint2*>(w)[i] = __ldg(reinterpret_cast<const uint2*>(src) + i);
    } else if (left > 0) {
      X* e = reinterpret_cast<X*>(w);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) e[j] = src[j];
    }
  }
  __device__ __forceinline__ float operator[](int j) const { return to_f32<X>(reinterpret_cast<const X*>(w)[j]); }
};
__device__ __forceinline__ bool finite_bits(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
// What whole numbers of units (a power of two, 1 / unit another) leave of v, exactly; all of it for infinities and NaN
__device__ __forceinline__ float rest_of(float v, float per_unit, float unit) {
  const float t = v * per_unit, n = rintf(t);
  return n == 0.f || !finite_bits(v) ? v : (t - n) * unit;
}

// NT: tiles of 8 columns (digits of rows).  GPS: groups per step.
//
// A CTA owns a run of row tiles; their (tile, unit of k) pairs are one list that the warps split evenly, so
// no warp waits for another until the end.  A warp streams its run through a ring of its own, filled by one
// lane's bulk copies.  Its part of a tile goes to shared memory when the tile ends, and the sums over warps
// are taken in their order at the end.
template <typename X, int NT, int GPS, bool ZERO>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_stream_kernel(const W4Params p) {
  using D = Digits<X, NT>;
  constexpr int ND = D::N;
  constexpr int COLS = 8 * NT;
  constexpr int SB = GPS * 16 * static_cast<int>(sizeof(X));  // scale bytes of a step
  constexpr int ZB = ZERO ? GPS * 16 : 0;
  constexpr int kUnit = unit_of(SB + ZB);
  constexpr int REC = kStepBytes + SB + ZB;
  constexpr int STAGE = kUnit * REC;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint64_t bars[kWarps][kDepth];
  __shared__ int abort_flag, kept;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nrow = p.rows, ncol = nrow * ND;
  const int pitch = p.chunk_steps * 128 + 16;  // bytes of a column
  unsigned char* ring = smem;
  float* red = reinterpret_cast<float*>(smem + kWarps * kDepth * STAGE);
  // of a group and two neighbouring columns: where their sums start (ZERO: the sums of the digits), their units
  int4* start = reinterpret_cast<int4*>(red + (p.tpb + kWarps - 1) * 16 * COLS);  // [group][COLS / 2]
  unsigned char* xs = reinterpret_cast<unsigned char*>(start + p.chunk_steps * GPS * COLS / 2);  // [column][step][q][b][8]
  uint16_t* marks = reinterpret_cast<uint16_t*>(xs + ncol * pitch);               // [step][kMarkRows]
  float* rest_at = reinterpret_cast<float*>(marks + p.chunk_steps * kMarkRows);  // [block][32]
  bool rests = false;  // whether the chunk has any
  // A thread's first items of x, eight values each, are on their way before the codes: behind those they
  // would wait for as long as the copies in flight take (3 us measured)
  const int sr = div_by(warp, p.by_wpr), si = (warp - sr * p.wpr) * 32 + lane, sn = p.wpr * 32;
  const X* x = static_cast<const X*>(p.x);
  const X* xr = x + sr * p.ldx;
  const int x_steps = min(p.chunk_steps, p.g.steps);
  auto load_x = [&](Raw8<X>& v, int s0, int ns, int i) {
    v.load(xr + s0 * 128 + i * 8, sr < nrow && i < ns * 16 ? p.K - s0 * 128 - i * 8 : 0, p.align);
  };
  Raw8<X> x0, x1;
  load_x(x0, 0, x_steps, si);
  load_x(x1, 0, x_steps, si + sn);
  if (tid == 0) abort_flag = kept = 0;
  if (lane == 0) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) mbar_init(&bars[warp][d], 1);
    fence_mbar_init();
  }
  __syncthreads();
  const WaitCtx wait{p.status, &abort_flag};

  const int t_lo = p.tiles_q * blockIdx.x + min(static_cast<int>(blockIdx.x), p.tiles_r);
  const int t_hi = t_lo + p.tiles_q + (static_cast<int>(blockIdx.x) < p.tiles_r ? 1 : 0);
  const int chunks = p.chunks;
  const int spt = p.chunk_steps;  // steps a tile has in a chunk, the same in every chunk (the last one's surplus is
                                  // skipped), so that a warp's tiles are too
  const int g = lane >> 2, q = lane & 3;
  unsigned char* myring = ring + warp * kDepth * STAGE;
  uint32_t phase = 0;  // of each stage's barrier, one bit a stage
  bool ok = true;

  for (int tb = t_lo; tb < t_hi; tb += p.tpb) {
    const int nt = min(p.tpb, t_hi - tb);
    const int total = nt * spt;
    const int per = (total + kWarps - 1) / kWarps;  // steps of a warp
    const int f_lo = min(total, warp * per), f_hi = min(total, f_lo + per);
    for (int ch = 0; ch < chunks; ++ch) {
      const int s0 = ch * p.chunk_steps;
      const int ns = min(p.chunk_steps, p.g.steps - s0);
      // The copies follow the warp's steps in memory: with x in one chunk its whole run is contiguous, else
      // the part of each tile.  `is` is the step of the tile, `fi` the place in the list.
      const bool whole = chunks == 1;
      const int tile_lo = div_by(f_lo, p.by_steps), step_lo = f_lo - tile_lo * spt;
      int is = step_lo, fi = f_lo, ist = 0;
      auto copy_len = [&](int f, int st) { return min(min(kUnit, f_hi - f), whole ? kUnit : ns - st); };
      const long long first = static_cast<long long>(tb + tile_lo) * p.g.steps + s0 + is;
      const unsigned char* src = p.data + first * REC;
      auto issue = [&]() {
        if (!whole && is >= ns) {  // on to the next tile
          src += (p.g.steps - is) * REC;
          fi += spt - is;
          is = 0;
        }
        if (fi >= f_hi || !ok) return;
        const int n = copy_len(fi, is);
        if (lane == 0) {
          uint64_t* bar = &bars[warp][ist];
          mbar_arrive_expect_tx(bar, n * REC);
          bulk_load(myring + ist * STAGE, src, n * REC, bar);
        }
        ist = ist + 1 == kDepth ? 0 : ist + 1;
        fi += n;
        is += n;
        src += n * REC;
      };
#pragma unroll
      for (int d = 0; d < kDepth; ++d) issue();

      if ((tb == t_lo && ch == 0) || !whole) {
        if (ch > 0 || tb > t_lo) {
          __syncthreads();  // the chunk before is no longer read
          if (rests) {
            if (tid == 0) kept = 0;
            __syncthreads();
          }
          load_x(x0, s0, ns, si);
          load_x(x1, s0, ns, si + sn);
        }
        const int items = (ns * 16 + 31) / 32 * 32;  // whole warps, since lanes share a step
        bool any_rest = false;
#pragma unroll 1
        for (int i = sr < nrow ? si : items; i < items; i += sn) {
          const Raw8<X> raw = x0;
          x0 = x1;
          load_x(x1, s0, ns, i + 2 * sn);
          float v[8], least = INFINITY;
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = raw[j];
            m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
          }
          if (__any_sync(0xffffffffu, m >= 0x7f800000u)) {
            m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] = finite_bits(v[j]) ? v[j] : 0.f;
              m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
            }
          }
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const int e = max(static_cast<int>((m + kRoundUp) >> 23), D::bits);
          const float up = __uint_as_float(static_cast<uint32_t>(D::top + 126 - e + 127) << 23);
          uint32_t w[8], wl[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // the bytes of (n + B) ^ B are the balanced digits of n (B has 0x80 in every byte but the top one)
            constexpr uint32_t B = D::H == 4 ? 0x808080u : 0x8080u, BL = D::L == 3 ? 0x8080u : 0x80u;
            least = fminf(least, fabsf(v[j]));
            const float t = v[j] * up;
            const int n = __float2int_rn(t);
            w[j] = (static_cast<uint32_t>(n) + B) ^ B;
            if (D::L) wl[j] = (static_cast<uint32_t>(__float2int_rn((t - static_cast<float>(n)) * (1 << D::low))) + BL) ^ BL;
          }
          const int st = i >> 4, b = (i >> 2) & 3, iq = i & 3;
          const bool live = i < ns * 16;
          const int unit0 = e + 1 - D::bits;  // exponent bits of 2^(e - 126 - bits)
          // all bits of a value from 2^(e - 126 - bits + precision - 1) on are whole units
          const float whole = __uint_as_float(static_cast<uint32_t>(unit0 + kPrecision<X> - 1) << 23);
          uint32_t mark = 0;
          if (__any_sync(0xffffffffu, live && least < whole)) {
            const float unit = __uint_as_float(static_cast<uint32_t>(unit0) << 23);
            const float per_unit = __uint_as_float(static_cast<uint32_t>(254 - unit0) << 23);
            bool rest = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] = rest_of(raw[j], per_unit, unit);
              rest |= v[j] != 0.f;
            }
            uint32_t with = __ballot_sync(0xffffffffu, rest) >> (lane & 16);  // four lanes a block
            with |= with >> 2;
            with = (with | with >> 1) & 0x1111u;
            with = (with | with >> 3 | with >> 6 | with >> 9) & 15u;
            int at = 0;  // the order in which rows and steps come here changes where the rests are, and nothing else
            if (with && (lane & 15) == 0) at = atomicAdd(&kept, __popc(with));
            at = __shfl_sync(0xffffffffu, at, lane & 16);
            const bool fits = at + 4 <= p.keep;
            mark = with | (fits ? at << 4 : 0xfff0);
            if (fits && (with >> b & 1)) {
              float* to = rest_at + (at + __popc(with & ((1u << b) - 1))) * 32 + iq * 8;
#pragma unroll
              for (int j = 0; j < 8; ++j) to[j] = v[j];
            }
            any_rest |= with != 0;
          }
          if (live && (lane & 15) == 0) marks[st * kMarkRows + sr] = mark;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            constexpr int L = D::L;
            const uint32_t(&wd)[8] = d < L ? wl : w;
            const uint32_t sel = 0x0040u + 0x0011u * (d < L ? d : d - L);  // that byte of each, and 4 bytes on
            const uint32_t lo = __byte_perm(__byte_perm(wd[0], wd[1], sel), __byte_perm(wd[2], wd[3], sel), 0x5410);
            const uint32_t hi = __byte_perm(__byte_perm(wd[4], wd[5], sel), __byte_perm(wd[6], wd[7], sel), 0x5410);
            const int col = sr * ND + d;
            if (live) *reinterpret_cast<uint2*>(xs + col * pitch + st * 128 + iq * 32 + b * 8) = make_uint2(lo, hi);
            int sum = __dp4a(static_cast<int>(lo), 0x01010101, __dp4a(static_cast<int>(hi), 0x01010101, 0));
#pragma unroll
            for (int o = 1; o < 16 / GPS; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (live && (i & (16 / GPS - 1)) == 0) {
              int* at = reinterpret_cast<int*>(start + (i / (16 / GPS)) * (COLS / 2) + (col >> 1)) + (col & 1);
              at[0] = ZERO ? sum : kMagicBits - 8 * sum;
              at[2] = (unit0 + (d < L ? 8 * d : D::low + 8 * (d - L))) << 23;
            }
          }
        }
        rests = __syncthreads_or(any_rest);
      }

      int ct = tile_lo, cs = step_lo, cst = 0;
      // columns past the last hold what nobody reads
      const unsigned char* xl[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) xl[n] = xs + min(n * 8 + g, ncol - 1) * pitch + q * 32;
      const int4* sl = start + q;
      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
      auto flush = [&]() {
        // this warp's part of the tile: tiles and warps grow together along the list, so tile + warp is a
        // slot of its own
        float* slot = red + static_cast<size_t>(ct + warp) * 16 * COLS + g * COLS + 2 * q;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float2* d0 = reinterpret_cast<float2*>(slot + n * 8);
          float2* d1 = reinterpret_cast<float2*>(slot + 8 * COLS + n * 8);
          *d0 = ch == 0 ? make_float2(acc[n][0], acc[n][1]) : make_float2(d0->x + acc[n][0], d0->y + acc[n][1]);
          *d1 = ch == 0 ? make_float2(acc[n][2], acc[n][3]) : make_float2(d1->x + acc[n][2], d1->y + acc[n][3]);
          acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        }
      };
      // Adds the rests of row m in step cs, whose record is `rec`: a lane has the codes of eight k of each block
      auto add_rest = [&](const unsigned char* rec, int m, uint32_t mark) {
        const int col = m * ND;
        const float* at = rest_at + (mark >> 4) * 32 + q * 8;
        const bool in_memory = mark >> 4 != 0xfff;
        const int k0 = (s0 + cs) * 128 + q * 8;
        const X* sc = reinterpret_cast<const X*>(rec + kStepBytes) + g;
        float p0 = 0.f, p1 = 0.f;
#pragma unroll 1
        for (uint32_t blocks = mark & 15u; blocks; blocks &= blocks - 1) {
          const int b = __ffs(blocks) - 1;
          float r[8];
          if (in_memory) {
            const float4 lo = *reinterpret_cast<const float4*>(at), hi = *reinterpret_cast<const float4*>(at + 4);
            r[0] = lo.x, r[1] = lo.y, r[2] = lo.z, r[3] = lo.w;
            r[4] = hi.x, r[5] = hi.y, r[6] = hi.z, r[7] = hi.w;
            at += 32;
          } else {  // from x again
            const int4 first = start[cs * GPS * (COLS / 2) + (col >> 1)];
            const uint32_t unit = static_cast<uint32_t>(col & 1 ? first.w : first.z);
            Raw8<X> v;
            v.load(x + m * p.ldx + k0 + b * 32, p.K - k0 - b * 32, p.align);
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = rest_of(v[j], __uint_as_float((254u << 23) - unit), __uint_as_float(unit));
          }
          uint32_t w0 = *reinterpret_cast<const uint32_t*>(rec + lane * 16 + b * 4);
          uint32_t w1 = *reinterpret_cast<const uint32_t*>(rec + 512 + lane * 16 + b * 4);
          const int gi = b * GPS / 4 * 16;
          const float z0 = 8388608.f + (ZERO ? rec[kStepBytes + SB + gi + g] & 15 : 8);
          const float z1 = 8388608.f + (ZERO ? rec[kStepBytes + SB + gi + 8 + g] & 15 : 8);
          float c0 = 0.f, c1 = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {  // a code as the low byte of 2^23 is 2^23 + code
            if (j == 4) w0 >>= 4, w1 >>= 4;
            const uint32_t sel = 0x7650u + (j & 3);
            c0 = fmaf(__uint_as_float(__byte_perm(w0 & 0x0f0f0f0fu, 0x4b000000u, sel)) - z0, r[j], c0);
            c1 = fmaf(__uint_as_float(__byte_perm(w1 & 0x0f0f0f0fu, 0x4b000000u, sel)) - z1, r[j], c1);
          }
          p0 = fmaf(to_f32<X>(sc[gi]), c0, p0);
          p1 = fmaf(to_f32<X>(sc[gi + 8]), c1, p1);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          p0 += __shfl_xor_sync(0xffffffffu, p0, o);
          p1 += __shfl_xor_sync(0xffffffffu, p1, o);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {  // to the row's first column
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool here = n * 8 + 2 * q + h == col;
            acc[n][h] += here ? p0 : 0.f;
            acc[n][2 + h] += here ? p1 : 0.f;
          }
        }
      };
      int f = f_lo;
      if (cs >= ns) {  // starts in the last chunk's surplus
        f += spt - cs;
        cs = 0;
        ++ct;
      }
      while (f < f_hi) {
        const int n_steps = copy_len(f, cs);
        ok = mbar_wait_w(&bars[warp][cst], (phase >> cst) & 1u, wait);
        if (!ok) break;
        phase ^= 1u << cst;
        const unsigned char* stg = myring + cst * STAGE;
        auto step = [&](int u) {
          const unsigned char* rec = stg + u * REC;
          const uint4 w0 = *reinterpret_cast<const uint4*>(rec + lane * 16);
          const uint4 w1 = *reinterpret_cast<const uint4*>(rec + 512 + lane * 16);
          const uint32_t wa[4] = {w0.x, w0.y, w0.z, w0.w}, wb[4] = {w1.x, w1.y, w1.z, w1.w};
          const X* sc = reinterpret_cast<const X*>(rec + kStepBytes) + g;
          const unsigned char* zp = rec + kStepBytes + SB + g;
          uint32_t xb[NT][8];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 x0 = *reinterpret_cast<const uint4*>(xl[n] + cs * 128);
            const uint4 x1 = *reinterpret_cast<const uint4*>(xl[n] + cs * 128 + 16);
            xb[n][0] = x0.x, xb[n][1] = x0.y, xb[n][2] = x0.z, xb[n][3] = x0.w;
            xb[n][4] = x1.x, xb[n][5] = x1.y, xb[n][6] = x1.z, xb[n][7] = x1.w;
          }
          int part[NT][4];
          int4 begin[NT];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            constexpr int BPG = 4 / GPS;  // blocks of a group
            const int gr = cs * GPS + b / BPG;
            if (b % BPG == 0) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                begin[n] = sl[gr * (COLS / 2) + n * 4];
                part[n][0] = part[n][2] = ZERO ? kMagicBits : begin[n].x;
                part[n][1] = part[n][3] = ZERO ? kMagicBits : begin[n].y;
              }
            }
            const uint32_t a[4] = {wa[b] & 0x0f0f0f0fu, wb[b] & 0x0f0f0f0fu, (wa[b] >> 4) & 0x0f0f0f0fu,
                                   (wb[b] >> 4) & 0x0f0f0f0fu};
#pragma unroll
            for (int n = 0; n < NT; ++n) imma16832(part[n], a, xb[n][2 * b], xb[n][2 * b + 1]);
            if (b % BPG == BPG - 1) {
              const float s0f = to_f32<X>(sc[(b / BPG) * 16]), s1f = to_f32<X>(sc[(b / BPG) * 16 + 8]);
              float z0 = 0.f, z1 = 0.f;
              if (ZERO) {
                z0 = -static_cast<float>(zp[(b / BPG) * 16] & 15u);
                z1 = -static_cast<float>(zp[(b / BPG) * 16 + 8] & 15u);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __int_as_float(part[n][e]) - kMagic;
                if (ZERO) {
                  const float d0 = static_cast<float>(begin[n].x), d1 = static_cast<float>(begin[n].y);
                  v[0] = fmaf(z0, d0, v[0]);
                  v[1] = fmaf(z0, d1, v[1]);
                  v[2] = fmaf(z1, d0, v[2]);
                  v[3] = fmaf(z1, d1, v[3]);
                }
                const float u0 = __int_as_float(begin[n].z), u1 = __int_as_float(begin[n].w);
                acc[n][0] = fmaf(s0f * u0, v[0], acc[n][0]);
                acc[n][1] = fmaf(s0f * u1, v[1], acc[n][1]);
                acc[n][2] = fmaf(s1f * u0, v[2], acc[n][2]);
                acc[n][3] = fmaf(s1f * u1, v[3], acc[n][3]);
              }
            }
          }
        };
#pragma unroll 2
        for (int u = 0; u < n_steps; ++u) {
          step(u);
          if (rests) {
            const uint32_t mark = lane < nrow ? marks[cs * kMarkRows + lane] : 0;
            for (uint32_t rows = __ballot_sync(0xffffffffu, mark != 0); rows; rows &= rows - 1) {
              const int m = __ffs(rows) - 1;
              add_rest(stg + u * REC, m, __shfl_sync(0xffffffffu, mark, m));
            }
          }
          ++f;
          if (++cs == ns) {
            flush();
            f += spt - ns;
            cs = 0;
            ++ct;
          }
        }
        __syncwarp();  // the stage has been read
        issue();
        cst = cst + 1 == kDepth ? 0 : cst + 1;
      }
      if (cs > 0) flush();
    }
    if (!ok) {  // a copy never came (its time limit has passed): wait for those in flight, then leave
#pragma unroll
      for (int d = 0; d < kDepth; ++d) mbar_drain(&bars[warp][d], (phase >> d) & 1u);
    }
    __syncthreads();
    // Sums over the warps that had a part of a tile, in their order; then over the digits
    const int log_rows = p.gated ? 3 : 4, orow = 1 << log_rows;
    for (int i = tid; i < nt * orow * nrow; i += kWarps * 32) {
      const int r = i & (orow - 1), tm = i >> log_rows;
      const int t = div_by(tm, p.by_rows), m = tm - t * nrow;
      const int n = (tb + t) * orow + r;
      if (n >= (p.gated ? p.N / 2 : p.N)) continue;
      float s[2][ND];
#pragma unroll
      for (int d = 0; d < ND; ++d) s[0][d] = s[1][d] = 0.f;
      // the warps that have the tile's first and last step
      const int w_lo = static_cast<unsigned>(t * spt) / static_cast<unsigned>(per);
      const int w_hi = static_cast<unsigned>((t + 1) * spt - 1) / static_cast<unsigned>(per);
#pragma unroll 4
      for (int w = w_lo; w <= w_hi; ++w) {
        const float* slot = red + (t + w) * 16 * COLS + r * COLS + m * ND;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          s[0][d] += slot[d];
          if (p.gated) s[1][d] += slot[8 * COLS + d];
        }
      }
      float out[2] = {0.f, 0.f};
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        out[0] += s[0][d];
        out[1] += s[1][d];
      }
      if (p.gated) out[0] = out[0] / (1.f + expf(-out[0])) * out[1];
      static_cast<X*>(p.y)[m * p.ldy + n] = from_f32<X>(out[0]);
    }
    __syncthreads();
  }
}

template <typename X, int NT, int GPS, bool ZERO>
int launch_stream(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows, int* status,
                  cudaStream_t st) {
  using D = Digits<X, NT>;
  constexpr int ND = D::N;
  constexpr int COLS = 8 * NT;
  constexpr int SIDE = GPS * 16 * static_cast<int>(sizeof(X)) + (ZERO ? GPS * 16 : 0);
  constexpr int kUnit = unit_of(SIDE);
  constexpr int STAGE = kUnit * (kStepBytes + SIDE);
  W4Params p;
  p.data = static_cast<const unsigned char*>(w->data);
  p.x = x;
  p.y = y;
  p.ldx = ldx;
  p.ldy = ldy;
  p.status = status;
  p.rows = rows;
  p.N = w->N;
  p.K = w->K;
  p.gated = w->gated;
  p.g = w4_geom(w);
  const uintptr_t starts = reinterpret_cast<uintptr_t>(x) | (rows > 1 ? static_cast<uintptr_t>(ldx) * sizeof(X) : 0);
  p.align = starts % 16 == 0 ? 16 : starts % 8 == 0 ? 8 : 2;
  const int ccols = rows * ND;
  const int grid = std::min(p.g.tiles, 148);
  p.tpb = std::min(NT > 2 ? 4 : 16, (p.g.tiles + grid - 1) / grid);
  const int fixed = kWarps * kDepth * STAGE + (p.tpb + kWarps - 1) * 16 * COLS * 4;
  // x of as many steps as fit, in chunks of one length
  const int per_step = ccols * 128 + GPS * COLS * 8 + kMarkRows * 2;
  const int room = kMaxSmem - 2048 - fixed - ccols * 16;
  const int fit = (room - 32 * 128) / per_step / kUnit * kUnit;  // beside 32 blocks of rests
  if (fit < kUnit) return KATA_ERR_UNSUPPORTED;
  const int chunks = (p.g.steps + fit - 1) / fit;
  p.tiles_q = p.g.tiles / grid;
  p.tiles_r = p.g.tiles % grid;
  p.wpr = kWarps / rows;
  p.by_rows = recip(rows);
  p.by_wpr = recip(p.wpr);
  p.chunk_steps = chunks == 1 ? p.g.steps : ((p.g.steps + chunks - 1) / chunks + kUnit - 1) / kUnit * kUnit;
  p.chunks = (p.g.steps + p.chunk_steps - 1) / p.chunk_steps;
  p.by_steps = recip(p.chunk_steps);
  p.keep = std::min(kMaxRests, (room - p.chunk_steps * per_step) / 128);
  const size_t smem = fixed + static_cast<size_t>(p.chunk_steps) * per_step + ccols * 16 + p.keep * 128;
  auto kern = w4_stream_kernel<X, NT, GPS, ZERO>;
  static std::atomic<uint64_t> allowed{0};
  if (int e = allow_smem(reinterpret_cast<const void*>(kern), kMaxSmem - 2048, allowed)) return e;
  kern<<<grid, kWarps * 32, smem, st>>>(p);
  return from_cuda(cudaGetLastError());
}

template <typename X, int NT>
int launch_groups(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows,
                  int* status, cudaStream_t st) {
  const int gps = w->group < 128 ? 128 / w->group : 1;
  if (w->zeros) {
    if (gps == 4) return launch_stream<X, NT, 4, true>(w, x, ldx, y, ldy, rows, status, st);
    if (gps == 2) return launch_stream<X, NT, 2, true>(w, x, ldx, y, ldy, rows, status, st);
    return launch_stream<X, NT, 1, true>(w, x, ldx, y, ldy, rows, status, st);
  }
  if (gps == 4) return launch_stream<X, NT, 4, false>(w, x, ldx, y, ldy, rows, status, st);
  if (gps == 2) return launch_stream<X, NT, 2, false>(w, x, ldx, y, ldy, rows, status, st);
  return launch_stream<X, NT, 1, false>(w, x, ldx, y, ldy, rows, status, st);
}

template <typename X>
int launch_rows(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows,
                int* status, cudaStream_t st) {
  if (rows <= Digits<X, 1>::rows()) return launch_groups<X, 1>(w, x, ldx, y, ldy, rows, status, st);
  if (rows <= Digits<X, 2>::rows()) return launch_groups<X, 2>(w, x, ldx, y, ldy, rows, status, st);
  if constexpr (sizeof(X) == 4) {
    if (rows > Digits<X, 3>::rows()) return launch_groups<X, 4>(w, x, ldx, y, ldy, rows, status, st);
  }
  return launch_groups<X, 3>(w, x, ldx, y, ldy, rows, status, st);
}

// ------------------------------------------------------------------------------------------------
// Tensor-core kernel: more rows than that.
//
// The weight is the A operand: 128 of its rows (8 tiles) by a step of 128 k, turned to 16-bit floats by the
// unpack warps straight into tensor memory (a row is a TMEM lane, so a thread unpacks words of its own
// row), and x the B operand by TMA: nothing of A passes through shared memory, whose bandwidth B needs.
// Codes to floats: a code as a byte beside 0x43 (0x64) is 128 + code in bf16 (1024 + code in f16), and one
// fused multiply-add leaves unit (code - zero), exactly.  With bf16 the unit is 2^-11: a step's sum, of at most
// 128 times 15 units of x, stays finite for every finite x; the scale takes it back.  fp32 x is three bf16 parts, each a column.
//
// A group's products go to one of 2 or 4 accumulators; the drain warps add it, times the rows' scales, to
// fp32 registers while another one fills, so that scales stay exact.  Unpacking and draining have warps of
// their own: in one loop each waits for what the other has just started (1750 cycles a step measured).
// With few row blocks a cluster's CTAs split k and add their sums through shared memory.
//
// Measured (device time): 8 to 32 x 8192 x 8192 in 23.8 us, 8 x 8192 x 32768 in 74.9 us (two rounds of 256 row blocks on
// 148 SMs), 64 x 4096 x 16384 gated in 27.5 us, 512 x 4096 x 4096 in 34.4 us (500 TFLOP/s) and 2048 in 130 us; fp32
// 64 x 4096 x 4096 in 18.4 us, 512 in 74.4 us.  Bound by issue: the unpack warps' 11 instructions a word, and the MMA warp, which takes
// 750 cycles for a step's 8 MMAs beside them, whatever their width.
// ------------------------------------------------------------------------------------------------

template <typename T>
struct Magic;
template <>
struct Magic<__nv_bfloat16> {
  static constexpr uint32_t base = 0x43434343u;
  static constexpr float back = 2048.f;
  static __device__ __forceinline__ uint32_t offset(uint32_t zero) {  // -(128 + zero) 2^-11
    const __nv_bfloat162 v = __float2bfloat162_rn(-(128.f + static_cast<float>(zero)) * (1.f / 2048.f));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b) {
    const uint32_t u = 0x3a003a00u;  // 2^-11
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&u),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Magic<__half> {
  static constexpr uint32_t base = 0x64646464u;
  static constexpr float back = 1.f;
  static __device__ __forceinline__ uint32_t offset(uint32_t zero) { return 0xe400e400u + 0x00010001u * zero; }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b) {
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
// The eight codes of a word, in order, as four pairs
template <typename T>
__device__ __forceinline__ void unpack8(uint32_t word, uint32_t offset, uint32_t* out) {
  const uint32_t lo = word & 0x0f0f0f0fu, hi = (word >> 4) & 0x0f0f0f0fu;
  out[0] = Magic<T>::fma2(__byte_perm(lo, Magic<T>::base, 0x4140), offset);
  out[1] = Magic<T>::fma2(__byte_perm(lo, Magic<T>::base, 0x4342), offset);
  out[2] = Magic<T>::fma2(__byte_perm(hi, Magic<T>::base, 0x4140), offset);
  out[3] = Magic<T>::fma2(__byte_perm(hi, Magic<T>::base, 0x4342), offset);
}

// An fp32 value as three bf16 parts, each the leading 8 bits of what is left: exact together (but for bits below
// 2^-133, which bf16 does not have: of values from 2^-110 on nothing), and no part overflows.  Infinities and NaN stay in the first part.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  const float a = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const bool fin = finite_bits(x);
  const float r = fin ? x - a : 0.f;
  const float b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  p[0] = __float2bfloat16_rn(fin ? a : x);
  p[1] = __float2bfloat16_rn(b);
  p[2] = __float2bfloat16_rn(r - b);
}

// x in the form that TMA takes: [part][row][ld], ld a multiple of 8 (fp32 rows as their parts, 16-bit rows that
// do not lie on 16-byte boundaries as they are)
template <typename T, typename X>
__global__ void __launch_bounds__(256) w4_parts_kernel(const X* __restrict__ x, long long ldx, T* __restrict__ out, long long rows,
                                                       int K, int ld) {
  const long long n = rows * ld;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const long long r = i / ld;
    const int k = static_cast<int>(i - r * ld);
    const X v = k < K ? x[r * ldx + k] : from_f32<X>(0.f);
    if constexpr (sizeof(X) == 4) {
      __nv_bfloat16 p[3];
      split3(v, p);
#pragma unroll
      for (int c = 0; c < 3; ++c) out[c * n + i] = p[c];
    } else {
      out[i] = v;
    }
  }
}

__device__ __forceinline__ void tma_load_x(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(0)
      : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// n MMAs (4 or 2) along k inside one 64-column box of x, one election for all: the MMA warp shares its scheduler
// with busy warps, and every instruction it does not issue counts
template <int n>
__device__ __forceinline__ void umma_ts_chain(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (n == 4)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 b1;\n\t.reg .b32 a1;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "add.u64 b1, %2, 2;\n\tadd.u32 a1, %1, 8;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

struct GemmParams {
  const unsigned char* data;
  void* y;
  long long ldy;
  int* status;
  int rows, N, gated, zeros;
  W4Geom g;
  int cs;
};

// Warps: codes' copies, x's copies, MMAs, (an idle one,) 8 drain, 8 unpack.  A copy costs its warp 115 cycles, so codes come
// in runs of 4 steps of a tile and x has a warp of its own (one warp, a step at a time: 1430 cycles a step).
constexpr int kRun = 4;
constexpr int kCodeStages = 2;

template <int R, int PARTS>
struct GemmSmem {
  static constexpr int N = R * PARTS;
  static constexpr int UW = 8;  // unpack warps (16 slow the MMA warp down, which shares its scheduler: 27.9 against 24.7 us)
  static constexpr int threads = 32 * (12 + UW);
  static constexpr int XS = N <= 64 ? 6 : N <= 128 ? 4 : 2;  // stages of x, 128 k each
  static constexpr int REC = 1024 + 4 * 16 * (PARTS == 3 ? 5 : 3);
  static constexpr int AS = N <= 128 ? 4 : 2;  // TMEM: stages of A, 64 columns each,
  static constexpr int DS = N <= 64 ? 4 : 2;   // and accumulators of N columns
  unsigned char x[XS][2][N * 128];
  unsigned char codes[kCodeStages][8][kRun * REC];
  uint64_t c_full[kCodeStages], c_free[kCodeStages], x_full[XS], x_free[XS], a_full[AS], a_free[AS], d_full[DS], d_free[DS];
  uint32_t tmem;
  int abort;
};

template <typename T, typename X, int R>
__global__ void __launch_bounds__(GemmSmem<R, sizeof(X) == 4 ? 3 : 1>::threads, 1) w4_gemm_kernel(const __grid_constant__ CUtensorMap tmx, const GemmParams p) {
  constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
  constexpr int N = R * PARTS;
  constexpr int HALF = R / 2;  // rows of x a thread sums
  using S = GemmSmem<R, PARTS>;
  constexpr int XS = S::XS, AS = S::AS, DS = S::DS, UW = S::UW;
  static_assert(DS * N + AS * 64 <= 512, "TMEM columns");
  extern __shared__ unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw + (1024 - (smem_u32(raw) & 1023)) % 1024);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.cs > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int tile0 = blockIdx.x / p.cs * 8, ntile = min(8, p.g.tiles - tile0);
  const int row0 = blockIdx.y * R;
  const int k_lo = p.g.steps * rank / p.cs, ns = p.g.steps * (rank + 1) / p.cs - k_lo;
  const int gps = p.g.gps;
  if (tid == 0) {
    sm.abort = 0;
    for (int i = 0; i < kCodeStages; ++i) {
      mbar_init(&sm.c_full[i], 1);
      mbar_init(&sm.c_free[i], UW + 8);
    }
    for (int i = 0; i < XS; ++i) {
      mbar_init(&sm.x_full[i], 1);
      mbar_init(&sm.x_free[i], 1);
    }
    for (int i = 0; i < AS; ++i) {
      mbar_init(&sm.a_full[i], UW);
      mbar_init(&sm.a_free[i], 1);
    }
    for (int i = 0; i < DS; ++i) {
      mbar_init(&sm.d_full[i], 1);
      mbar_init(&sm.d_free[i], 8);
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem, tmem_a = tbase + DS * N;
  const WaitCtx wc{p.status, &sm.abort};
  float acc[HALF];
#pragma unroll
  for (int j = 0; j < HALF; ++j) acc[j] = 0.f;

  if (warp == 0) {
    // lane t copies the records of tile t
    const unsigned char* src = p.data + (static_cast<long long>(tile0 + lane) * p.g.steps + k_lo) * p.g.rec;
    int n = 0;  // runs copied
    for (; n * kRun < ns; ++n) {
      const int c = n % kCodeStages, bytes = min(kRun, ns - n * kRun) * p.g.rec;
      if (n >= kCodeStages && !mbar_wait_w(&sm.c_free[c], (n / kCodeStages - 1) & 1, wc)) break;
      if (lane == 0) mbar_arrive_expect_tx(&sm.c_full[c], ntile * bytes);
      __syncwarp();
      if (lane < ntile) bulk_load(sm.codes[c][lane], src, bytes, &sm.c_full[c]);
      src += bytes;
    }
    if (sm.abort) {  // copies in flight land before the CTA goes
      for (int i = max(0, n - kCodeStages); i < n; ++i) mbar_drain(&sm.c_full[i % kCodeStages], (i / kCodeStages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) tma_prefetch_desc(&tmx);
    int n = 0;
    for (; n < ns; ++n) {
      const int xs = n % XS;
      if (n >= XS && !mbar_wait_w(&sm.x_free[xs], (n / XS - 1) & 1, wc)) break;
      if (lane == 0) mbar_arrive_expect_tx(&sm.x_full[xs], 2 * N * 128);
      __syncwarp();
      if (lane < 2) tma_load_x(sm.x[xs][lane], &tmx, &sm.x_full[xs], (k_lo + n) * 128 + lane * 64, row0);
    }
    if (sm.abort) {
      for (int i = max(0, n - XS); i < n; ++i) mbar_drain(&sm.x_full[i % XS], (i / XS) & 1);
    }
    __syncwarp();
  } else if (warp == 2) {
    constexpr uint32_t idesc = umma_idesc_f16(128, N, std::is_same<T, __nv_bfloat16>::value, false, false);
    int gi = 0, s = 0;  // groups and steps issued
    const uint64_t bd0 = umma_smem_desc(smem_u32(sm.x[0][0]), 16, 1024, 128);
    auto issue = [&](auto gps_c) {  // the groups of a step as a constant: the issue path is one thread's
      constexpr int G = decltype(gps_c)::value;
      int xs = 0, as = 0, ds = 0;
      uint32_t xph = 0, aph = 0, dph = 1;  // phases of the barriers waited for
      for (; s < ns; ++s) {
        if (!mbar_wait_w(&sm.x_full[xs], xph, wc) || !mbar_wait_w(&sm.a_full[as], aph, wc)) return;
        tc_fence_after();
        const uint32_t a = tmem_a + as * 64;
        const uint64_t bd = bd0 + static_cast<uint64_t>(xs * (2 * N * 128 / 16));
#pragma unroll
        for (int g = 0; g < G; ++g, ++gi) {
          if (gi >= DS) {
            if (!mbar_wait_w(&sm.d_free[ds], dph, wc)) return;
            tc_fence_after();
          }
          constexpr int CH = G == 4 ? 2 : 4;
#pragma unroll
          for (int k = 0; k < 8 / G; k += CH) {
            const int kk = g * (8 / G) + k;
            umma_ts_chain<CH>(tbase + ds * N, a + 8 * kk, bd + static_cast<uint64_t>(((kk >> 2) * (N * 128) + (kk & 3) * 32) >> 4),
                              idesc, k > 0);
          }
          umma_commit_w(&sm.d_full[ds]);
          if (++ds == DS) {
            ds = 0;
            dph ^= 1;
          }
        }
        umma_commit_w(&sm.a_free[as]);
        umma_commit_w(&sm.x_free[xs]);
        if (++xs == XS) {
          xs = 0;
          xph ^= 1;
        }
        if (++as == AS) {
          as = 0;
          aph ^= 1;
        }
      }
    };
    if (gps == 1)
      issue(std::integral_constant<int, 1>());
    else if (gps == 2)
      issue(std::integral_constant<int, 2>());
    else
      issue(std::integral_constant<int, 4>());
    if (s < ns && s > 0) mbar_drain(&sm.x_free[(s - 1) % XS], ((s - 1) / XS) & 1);
  } else if (warp >= 12) {  // unpack: the words of a row's q = NQ h ..
    constexpr int NQ = 16 / UW;
    const int quad = warp & 3, h = (warp - 12) >> 2;
    const int tile = quad * 2 + (lane >> 4), r16 = lane & 15;
    const uint32_t a_at = tmem_a + (static_cast<uint32_t>(32 * quad) << 16) + h * (4 * NQ);
    const uint32_t words_at = (r16 >> 3) * 512 + (r16 & 7) * 64 + h * (16 * NQ);
    const uint32_t zeros_at = kStepBytes + gps * 16 * sizeof(X) + r16;
    uint4 wq[NQ];
    uint32_t zo[4];  // of the step's blocks of 32 k
    auto fetch = [&](int s) {  // the words of step s
      const int run = s / kRun, c = run % kCodeStages;
      if (s % kRun == 0 && !mbar_wait_w(&sm.c_full[c], (run / kCodeStages) & 1, wc)) return false;
      const unsigned char* rec = sm.codes[c][tile] + (s % kRun) * p.g.rec;
#pragma unroll
      for (int i = 0; i < NQ; ++i) wq[i] = *reinterpret_cast<const uint4*>(rec + words_at + 16 * i);
      if (p.zeros) {
#pragma unroll
        for (int b = 0; b < 4; ++b) zo[b] = Magic<T>::offset(rec[zeros_at + (b * gps >> 2) * 16] & 15u);
      }
      return true;
    };
#pragma unroll
    for (int b = 0; b < 4; ++b) zo[b] = Magic<T>::offset(8);
    bool ok = ns > 0 && fetch(0);
    for (int s = 0; ok && s < ns; ++s) {
      const int as = s % AS;
      if (s >= AS && !mbar_wait_w(&sm.a_free[as], (s / AS - 1) & 1, wc)) break;
      tc_fence_after();
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t v[4 * NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) unpack8<T>(b == 0 ? wq[i].x : b == 1 ? wq[i].y : b == 2 ? wq[i].z : wq[i].w, zo[b], v + 4 * i);
        tmem_st8(a_at + as * 64 + b * 16, v);
      }
      if (s % kRun == kRun - 1) arrive_warp(&sm.c_free[s / kRun % kCodeStages]);
      ok = s + 1 >= ns || fetch(s + 1);  // under the stores
      tmem_wait_st();
      tc_fence_before();
      arrive_warp(&sm.a_full[as]);
    }
  } else if (warp >= 4) {  // drain
    const int quad = warp & 3, h = (warp - 4) >> 2;
    const int tile = quad * 2 + (lane >> 4), r16 = lane & 15;
    const uint32_t d_at = tbase + (static_cast<uint32_t>(32 * quad) << 16) + h * HALF;
    int ds = 0;
    uint32_t dph = 0;
    for (int s = 0; s < ns; ++s) {
      const int run = s / kRun, c = run % kCodeStages;
      if (s % kRun == 0 && !mbar_wait_w(&sm.c_full[c], (run / kCodeStages) & 1, wc)) break;
      const X* sc = reinterpret_cast<const X*>(sm.codes[c][tile] + (s % kRun) * p.g.rec + kStepBytes) + r16;
      float scale[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) scale[i] = i < gps ? to_f32<X>(sc[i * 16]) * Magic<T>::back : 0.f;
      if (s % kRun == kRun - 1) arrive_warp(&sm.c_free[c]);
      bool ok = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= gps) break;
        if (!(ok = mbar_wait_w(&sm.d_full[ds], dph, wc))) break;
        tc_fence_after();
#pragma unroll
        for (int pt = 0; pt < PARTS; ++pt) {
#pragma unroll
          for (int c0 = 0; c0 < HALF; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(d_at + ds * N + pt * R + c0, v);
            tmem_wait_ld();
            if (pt == PARTS - 1 && c0 + 16 == HALF) {  // all read
              tc_fence_before();
              arrive_warp(&sm.d_free[ds]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c0 + j] = fmaf(scale[i], __uint_as_float(v[j]), acc[c0 + j]);
          }
        }
        if (++ds == DS) {
          ds = 0;
          dph ^= 1;
        }
      }
      if (!ok) break;
    }
  }
  __syncthreads();
  const bool good = sm.abort == 0;

  // The sums through shared memory, [row of x][128 rows of the weight] (every copy and product has ended): the
  // registers' code is unrolled, and what follows would be fetched once for each of them (20000 cycles measured)
  float* buf = reinterpret_cast<float*>(sm.x);
  if (warp >= 4 && warp < 12) {
#pragma unroll
    for (int j = 0; j < HALF; ++j) buf[(((warp - 4) >> 2) * HALF + j) * 128 + (warp & 3) * 32 + lane] = acc[j];
  }
  if (p.cs > 1)
    cluster_sync();
  else
    __syncthreads();
  if (warp < 16 && good) {
    const int wrow = (warp & 3) * 32 + lane, r = wrow & 15, t = tile0 + (wrow >> 4);
    const int n = p.gated ? t * 8 + r : t * 16 + r;
    const bool mine = p.gated ? r < 8 && n < p.N / 2 : n < p.N;
    const int m_hi = min(R * (rank + 1) / p.cs, p.rows - row0);
#pragma unroll 1
    for (int m = R * rank / p.cs + (warp >> 2); m < m_hi; m += 4) {
      float v = buf[m * 128 + wrow];
      if (p.cs > 1) {  // over the CTAs of the cluster, in their order
        const uint32_t at = smem_u32(buf + m * 128 + wrow);
        v = 0.f;
        for (int c = 0; c < p.cs; ++c) v += ld_cluster(mapa_shared(at, c));
      }
      if (p.gated) {  // the up row is eight lanes on
        const float up = __shfl_down_sync(0xffffffffu, v, 8);
        v = v / (1.f + expf(-v)) * up;
      }
      if (mine) static_cast<X*>(p.y)[(row0 + m) * p.ldy + n] = from_f32<X>(v);
    }
  }
  if (p.cs > 1) cluster_sync();  // nobody reads this CTA's sums any more
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tbase, 512);
}

// Whether x can be read by TMA as it lies
bool tma_ready(int dtype, const void* x, long long ldx) {
  return dtype != KATA_DTYPE_F32 && ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

template <typename T, typename X, int R>
int launch_gemm(const kata_w4_weight* w, const void* x, long long ldx, long long plane, void* y, long long ldy, int rows,
                int* status, cudaStream_t st) {
  constexpr int PARTS = sizeof(X) == 4 ? 3 : 1;
  GemmParams p;
  p.data = static_cast<const unsigned char*>(w->data);
  p.y = y;
  p.ldy = ldy;
  p.status = status;
  p.rows = rows;
  p.N = w->N;
  p.gated = w->gated;
  p.zeros = w->zeros;
  p.g = w4_geom(w);
  const int blocks = (p.g.tiles + 7) / 8, slabs = (rows + R - 1) / R;
  // CTAs that split k, as many as the GPU has room for, with two steps each at least
  p.cs = std::max(1, std::min(std::min(8, 148 / (blocks * slabs)), p.g.steps / 2));
  CUtensorMap tm;
  const uint64_t dims[3] = {static_cast<uint64_t>(w->K), static_cast<uint64_t>(rows), PARTS};
  const uint64_t str[2] = {static_cast<uint64_t>(ldx) * 2, static_cast<uint64_t>(PARTS == 1 ? ldx * rows : plane) * 2};
  const uint32_t box[3] = {64, R, PARTS};
  if (int e = encode_tmap_16bit(&tm, x, 3, dims, str, box, 128)) return e;
  auto kern = w4_gemm_kernel<T, X, R>;
  static std::atomic<uint64_t> allowed{0};
  const int smem = static_cast<int>(sizeof(GemmSmem<R, PARTS>)) + 1024;
  if (int e = allow_smem(reinterpret_cast<const void*>(kern), smem, allowed)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * p.cs, slabs);
  cfg.blockDim = dim3(GemmSmem<R, PARTS>::threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cs;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.cs > 1 ? 1 : 0;
  return from_cuda(cudaLaunchKernelEx(&cfg, kern, tm, p));
}

// More rows than the streaming kernel takes: x as it lies where TMA can read it, else through the workspace.
template <typename T, typename X>
int run_gemm(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy, int rows, void* ws,
             int* status, cudaStream_t st) {
  long long plane = 0;
  if (!tma_ready(w->dtype, x, ldx)) {
    const int ld = (w->K + 7) / 8 * 8;
    plane = static_cast<long long>(rows) * ld;
    const int grid = static_cast<int>(std::min<long long>(148 * 8, (plane + 255) / 256));
    w4_parts_kernel<T, X><<<grid, 256, 0, st>>>(static_cast<const X*>(x), ldx, static_cast<T*>(ws), rows, w->K, ld);
    x = ws;
    ldx = ld;
  }
  if (rows <= 32) return launch_gemm<T, X, 32>(w, x, ldx, plane, y, ldy, rows, status, st);
  if (sizeof(X) == 4 || rows <= 64) return launch_gemm<T, X, 64>(w, x, ldx, plane, y, ldy, rows, status, st);
  if constexpr (sizeof(X) == 2) return launch_gemm<T, X, 128>(w, x, ldx, plane, y, ldy, rows, status, st);
  return KATA_OK;
}

int w4_check(const kata_w4_weight* w) {
  if (!w) return KATA_ERR_INVALID;
  if (w->dtype != KATA_DTYPE_F32 && w->dtype != KATA_DTYPE_BF16 && w->dtype != KATA_DTYPE_F16) return KATA_ERR_DTYPE;
  if (w->N < 1 || w->K < 1 || w->N > (1 << 24) || w->K > (1 << 24)) return KATA_ERR_SHAPE;
  if (w->group != 32 && w->group != 64 && (w->group < 128 || w->group % 128)) return KATA_ERR_SHAPE;
  if ((w->gated != 0 && w->gated != 1) || (w->zeros != 0 && w->zeros != 1)) return KATA_ERR_INVALID;
  if (w->gated && w->N % 2) return KATA_ERR_SHAPE;
  return KATA_OK;
}

// Rows that are streamed over.  Up to two column tiles the streaming kernel is ahead whatever the size (5 x 8192 x 8192:
// 21.2 against 23.4 us; fp32, 3 rows: 22.7 against 27.4 us; 3 x 4100 x 5003, g 32, zeros: 13.1 against 18.4 us); up to
// three, four of fp32, only while a weight is small and the fixed cost counts (8 x 768 x 768: 5.5 against 6.5 us; 8 x
// 2048 x 2048: 7.7 against 11.5, 8 x 4096 x 4096: 14.3 against 11.0 us; fp32, 6 x 2048 x 2048: 11.4 against 13.8, 6 x
// 8192 x 8192: 50 against 28 us).  Four column tiles of 16-bit rows spill and are behind (10 x 768 x 768: 8.1 against 6.7 us).
int stream_rows(const kata_w4_weight* w) {
  const W4Geom g = w4_geom(w);
  const bool small = static_cast<long long>(g.tiles) * g.steps <= 4096;
  if (w->dtype == KATA_DTYPE_F32) return small ? Digits<float, 4>::rows() : Digits<float, 2>::rows();
  return small ? Digits<__half, 3>::rows() : Digits<__half, 2>::rows();
}
size_t w4_esize(int dtype) { return dtype == KATA_DTYPE_F32 ? 4 : 2; }
bool w4_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace kata

using namespace kata;

extern "C" size_t kata_w4_bytes(const kata_w4_weight* w) {
  if (w4_check(w)) return 0;
  const W4Geom g = w4_geom(w);
  return static_cast<size_t>(g.tiles) * g.steps * g.rec;
}

extern "C" int kata_w4_pack(const void* packed, const void* scales, const void* zeros, const kata_w4_weight* w,
                            kata_stream_t stream) {
  if (int e = w4_check(w)) return e;
  if (!packed || !scales || !w->data || (!zeros) != (!w->zeros)) return KATA_ERR_INVALID;
  if (!w4_al16(w->data)) return KATA_ERR_ALIGN;
  const W4Geom g = w4_geom(w);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int grid = static_cast<int>(std::min<long long>(148 * 8, (static_cast<long long>(g.tiles) * g.steps + 7) / 8));
  const uint32_t* pk = static_cast<const uint32_t*>(packed);
  const uint8_t* z = static_cast<const uint8_t*>(zeros);
  unsigned char* data = static_cast<unsigned char*>(const_cast<void*>(w->data));
  if (w->dtype == KATA_DTYPE_F32)
    w4_pack_kernel<uint32_t><<<grid, 256, 0, st>>>(pk, static_cast<const uint32_t*>(scales), z, data, w->N, w->K, w->group,
                                                   w->gated, g);
  else
    w4_pack_kernel<uint16_t><<<grid, 256, 0, st>>>(pk, static_cast<const uint16_t*>(scales), z, data, w->N, w->K, w->group,
                                                   w->gated, g);
  return from_cuda(cudaGetLastError());
}

extern "C" size_t kata_w4_workspace_bytes(const kata_w4_weight* w, const void* x, long long ldx, long long rows) {
  if (w4_check(w) || rows <= stream_rows(w) || tma_ready(w->dtype, x, ldx)) return 0;
  return static_cast<size_t>(rows) * ((w->K + 7) / 8 * 8) * (w->dtype == KATA_DTYPE_F32 ? 6 : 2);
}

extern "C" int kata_w4_linear(const kata_w4_weight* w, const void* x, long long ldx, void* y, long long ldy,
                              long long rows, void* workspace, size_t workspace_bytes, int* status,
                              kata_stream_t stream) {
  if (int e = w4_check(w)) return e;
  if (rows < 0 || rows > (1ll << 21)) return KATA_ERR_SHAPE;  // slabs of at least 32 rows are the grid's y
  if (rows == 0) return KATA_OK;
  if (!w->data || !x || !y) return KATA_ERR_INVALID;
  if (!w4_al16(w->data)) return KATA_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(x) % w4_esize(w->dtype) || reinterpret_cast<uintptr_t>(y) % w4_esize(w->dtype))
    return KATA_ERR_ALIGN;
  if (rows > 1 && (ldx < w->K || ldy < (w->gated ? w->N / 2 : w->N))) return KATA_ERR_SHAPE;
  const size_t need = kata_w4_workspace_bytes(w, x, ldx, rows);
  if (need && (!workspace || workspace_bytes < need)) return KATA_ERR_WORKSPACE;
  if (need && !w4_al16(workspace)) return KATA_ERR_ALIGN;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int n = static_cast<int>(rows);
  if (rows <= stream_rows(w)) {
    if (w->dtype == KATA_DTYPE_BF16) return launch_rows<__nv_bfloat16>(w, x, ldx, y, ldy, n, status, st);
    if (w->dtype == KATA_DTYPE_F16) return launch_rows<__half>(w, x, ldx, y, ldy, n, status, st);
    return launch_rows<float>(w, x, ldx, y, ldy, n, status, st);
  }
  if (w->dtype == KATA_DTYPE_BF16) return run_gemm<__nv_bfloat16, __nv_bfloat16>(w, x, ldx, y, ldy, n, workspace, status, st);
  if (w->dtype == KATA_DTYPE_F16) return run_gemm<__half, __half>(w, x, ldx, y, ldy, n, workspace, status, st);
  return run_gemm<__nv_bfloat16, float>(w, x, ldx, y, ldy, n, workspace, status, st);
}
