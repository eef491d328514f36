// W8A8 linear layer with its epilogue: y = act((xq . w^T) * xs * ws + bias) + residual, for
// any token count (s8b_linear_w8a8).
//
// Two forms, by their cost (few_rows below):
//  * few rows: the weights are most of the cost (1 byte read per 2 M operations), so the decode
//    GEMM of gemm_tc.cu streams them with its K range split over CTAs, its int32 partials stay
//    in L2, and linear_epilogue_kernel sums, scales and finishes them;
//  * many rows: the product is bound by the int8 tensor pipe. linear_tc_kernel below tiles it
//    128 tokens x NT weight rows.
//
// linear_tc_kernel: one persistent CTA per SM walks output tiles. Warp 0 issues the TMA loads
// (128-byte K slices, 128B swizzle, a ring of kStages stages), one thread of warp 1 issues
// tcgen05.mma kind::i8 into one of two TMEM accumulators, and warps 2-9 finish the other
// accumulator meanwhile, so the epilogue costs time only where a tile's K loop is shorter than
// it. The int32 sums are exact; the scales are two rounded binary32 products in the order of
// the framework's other GEMMs, so without bias, activation and residual the result equals
// s8b_gemm_w8a8's bit for bit. All later steps stay in binary32 and the output is rounded once.
//
// Measured (us, in a graph that repeats the call / by the call, beside the floor: bytes at 6.53 TB/s,
// int8 operations at twice the measured bf16 rate, 3.27 Pop/s): 8 x 4096 x 4096 with residual 8.4 /
// 15.8 (2.6; two launches that overlap. One, with the sums joined over a cluster and the
// epilogue there, took 9 to 10 us: it cannot start before the slowest CTA of a cluster);
// 4096 x 4096 x 4096 with bias and residual 77 / 88 (42; 1.8 / 1.6 Pop/s); 8192 x 12288 x 4096 with
// SiLU 361 / 429 (252; 2.3 / 1.9 Pop/s, the latter under the power cap); 999 x 5127 x 1040 with bias
// and GELU 29.6 / 28.9 (3.3). The large ones are bound by the operands' way from L2: 128 x 256
// tiles ask it for some 94 bytes per SM and cycle.
//
// The epilogue turns 32 rows x 16 columns of a warp at a time through shared memory: TMEM
// hands a lane one row, while global memory wants neighbouring lanes on neighbouring columns
// (row-per-lane stores fill half a 32-byte sector each and cost four times as many).
#include <cstring>

#include "common.cuh"
#include "tcgen05.cuh"

namespace s8b {
namespace {

using namespace tc;

enum { kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3, kActRelu = 4 };

// v * sigmoid(z): exp overflows to +inf for z below -88.7, where the product, 2.7e-37 there, is given
// as the limit 0 (1 / (1 + e) or e / (1 + e) of e = exp(-|z|) would hold it down to binary32's
// end, for 1 us of 30 at 999 x 5127 x 1040).
__device__ __forceinline__ float times_sigmoid(float v, float z) {
  return __fdiv_rn(v, 1.0f + __expf(-z));
}
// v Phi(v), Phi the normal distribution. Its lower half is h(|v|) = e^(x^2) erfc(x) e^(-x^2) / 2 with
// x = |v| / sqrt 2, whose relative precision holds to binary32's end, where (1 + erf) / 2 cancels (ten
// bits are left of it at v = -4, none at -5.6). e^(x^2) erfc(x) falls smoothly from 1 like 1 / x:
// in t = 1 / (1 + 0.37 x) it is t times a polynomial, here of degree 6, fitted to it over x in
// [0, 9.6] for the least largest relative error, 7.6e-7. With erfcf instead the ragged product
// (999 x 5127 x 1040) takes 34.8 us, with this 29.8.
__device__ __forceinline__ float times_phi(float v) {
  const float t = __fdividef(1.0f, fmaf(0.26162952184677124f, fabsf(v), 1.0f));
  float q = -0.07118100672960281f;
  q = fmaf(q, t, 0.2174852341413498f);
  q = fmaf(q, t, -0.09271273016929626f);
  q = fmaf(q, t, 0.158327117562294f);
  q = fmaf(q, t, 0.07647876441478729f);
  q = fmaf(q, t, 0.10741057991981506f);
  q = fmaf(q, t, 0.10419242829084396f);
  const float lower = q * t * __expf(-0.5f * v * v);
  return v * (v < 0.0f ? lower : 1.0f - lower);
}
__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == kActSilu) return times_sigmoid(v, v);
  if (act == kActGelu) return times_phi(v);
  // (1 + tanh u) / 2 = sigmoid(2 u), u = sqrt(2/pi) (v + 0.044715 v^3)
  if (act == kActGeluTanh)
    return times_sigmoid(v, 1.5957691216057308f * v * (1.0f + 0.044715f * v * v));
  if (act == kActRelu) return v < 0.0f ? 0.0f : v;  // NaN stays NaN
  return v;
}

// The same of N values, the choice made once for all of them.
template <int N>
__device__ __forceinline__ void apply_act(float (&v)[N], int act) {
#define S8B_ACT_CASE(A)                                 \
  case A:                                               \
    _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = apply_act(v[i], A); \
    break;
  switch (act) {
    S8B_ACT_CASE(kActSilu)
    S8B_ACT_CASE(kActGelu)
    S8B_ACT_CASE(kActGeluTanh)
    S8B_ACT_CASE(kActRelu)
    default: break;
  }
#undef S8B_ACT_CASE
}

struct LinArgs {
  const float *xs, *ws;
  const void *bias, *res;
  void *y;
  int32_t *status;
  int M, N, kc, act;
  int tiles_m, tiles_n;
  int vec;  // out, bias and residual rows keep 16-byte alignment
};

constexpr int kTileM = 128;
constexpr int kSlice = 128;       // K bytes per stage
constexpr int kEpiPitch = 20;     // floats per staged row of 16 (16-byte rows, no bank conflicts)

template <int NT, bool ACT>
struct LinLayout {
  // An activation is long in instructions and a warp waits on most of them: 16 warps finish a
  // tile sooner where its K loop does not hide it (999 x 5127 x 1040 with GELU: 39.5 -> 29.8 us;
  // 4096 x 4096 x 4096 with SiLU, whose loop does: 88.6 -> 90.0). They cost a stage of the ring, so
  // without an activation it stays at 8 (4096 cubed with bias and residual: 77.6 against 81.0),
  // and beside 256-wide tiles' stages their staging has no room.
  static constexpr int kEpiWarps = NT == 128 && ACT ? 16 : 8;
  static constexpr int kStages = NT == 256 ? 4 : ACT ? 5 : 6;
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kCols = 4 * NT / kEpiWarps;  // columns that an epilogue warp finishes
  static constexpr int kStageBytes = (kTileM + NT) * kSlice;
  static constexpr int kEpi = kStages * kStageBytes;                 // staging of the epilogue
  static constexpr int kHdr = kEpi + kEpiWarps * 32 * kEpiPitch * 4;  // barriers
  static constexpr int kSmem = 1024 + kHdr + 256;
  static constexpr int kTmemCols = 2 * NT;
};

// Tile t of the launch: bands of kBand token tiles, weight tiles outermost inside a band, so
// the CTAs that run together share few weight tiles and a band's tokens stay in L2.
constexpr int kBand = 16;
__device__ __forceinline__ void tile_at(int t, const LinArgs &a, int *m0, int *n0, int NT) {
  const int per = kBand * a.tiles_n;
  const int band = t / per, r = t - band * per;
  const int rows = min(kBand, a.tiles_m - band * kBand);
  const int n = r / rows;
  *m0 = (band * kBand + r - n * rows) * kTileM;
  *n0 = n * NT;
}

template <typename T, int NT, bool ACT>
__global__ void __launch_bounds__(LinLayout<NT, ACT>::kThreads, 1)
    linear_tc_kernel(const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_w, const LinArgs a) {
  using L = LinLayout<NT, ACT>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + L::kHdr);
  uint64_t *empty = full + kStages;
  uint64_t *acc_full = empty + kStages;  // [2]
  uint64_t *acc_empty = acc_full + 2;    // [2]
  uint64_t *drained = acc_empty + 2;
  uint32_t *tmem_base = reinterpret_cast<uint32_t *>(drained + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_base + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_base)), "r"(L::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], L::kEpiWarps);
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base;
  griddep_wait();
  const int tiles = a.tiles_m * a.tiles_n;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, ph = 0, issued = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        int m0, n0;
        tile_at(t, a, &m0, &n0, NT);
        for (int k = 0; k < a.kc; ++k) {
          if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, a.status)) {
            ok = false;
            break;
          }
          uint8_t *st = sm + s * L::kStageBytes;
          mbar_expect_tx(&full[s], L::kStageBytes);
          tma_load_2d(st, &map_x, k * kSlice, m0, &full[s]);
          tma_load_2d(st + kTileM * kSlice, &map_w, k * kSlice, n0, &full[s]);
          ++issued;
          if (++s == kStages) s = 0, ph ^= 1;
        }
      }
      // every copy has landed before the shared memory goes: the last issue of each stage
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_drain(&full[i % kStages], (i / kStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = i8_idesc(128, NT);
      int s = 0, ph = 0, q = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++q) {
        const int b = q & 1;
        if (!mbar_wait(&acc_empty[b], ((q >> 1) & 1) ^ 1, abort_flag, a.status)) break;
        tc_fence_after();
        for (int k = 0; k < a.kc; ++k) {
          if (!mbar_wait(&full[s], ph, abort_flag, a.status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t xd = sw128_desc(smem_u32(sm + s * L::kStageBytes));
          const uint64_t wd = sw128_desc(smem_u32(sm + s * L::kStageBytes + kTileM * kSlice));
#pragma unroll
          for (int j = 0; j < kSlice / 32; ++j)
            mma_i8(tmem + b * NT, xd + 2 * j, wd + 2 * j, idesc, (k | j) != 0);
          mma_commit(&empty[s]);
          if (++s == kStages) s = 0, ph ^= 1;
        }
        if (ok) mma_commit(&acc_full[b]);
      }
      // the products in flight read shared memory and write TMEM: let them end
      mma_commit(drained);
      mbar_drain(drained, 0);
    }
  } else {
    const int ew = warp - 2, quad = warp & 3, part = ew >> 2;
    float *stg = reinterpret_cast<float *>(sm + L::kEpi) + ew * 32 * kEpiPitch;
    const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.res);
    T *y = static_cast<T *>(a.y);
    constexpr int kCols = L::kCols;
    int q = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++q) {
      const int b = q & 1;
      int m0, n0;
      tile_at(t, a, &m0, &n0, NT);
      const bool ok = mbar_wait(&acc_full[b], (q >> 1) & 1, abort_flag, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const int mrow = m0 + 32 * quad;
      const float sx = mrow + lane < a.M ? a.xs[mrow + lane] : 0.0f;
      const uint32_t acc = tmem + b * NT + part * kCols + (static_cast<uint32_t>(32 * quad) << 16);
      const int nbase = n0 + part * kCols;
      // Columns of this warp that exist. While a chunk of 16 is finished from shared memory, the
      // next one's sums are on their way from TMEM and its residual from global memory (loaded
      // when needed, the residual cost 12 of 89 us at 4096 x 4096 x 4096).
      const int cols = mrow < a.M ? min(kCols, a.N - nbase) : 0;
      uint32_t v[16];
      uint4 rnext[2] = {};
      auto ask = [&](int c) {  // the residual of chunk c (vector rows)
        const int n = nbase + c + 8 * (lane & 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = mrow + (lane >> 1) + 16 * i;
          if (c < cols && n < a.N && m < a.M)
            rnext[i] = *reinterpret_cast<const uint4 *>(res + static_cast<size_t>(m) * a.N + n);
        }
      };
      float wnext = 0.0f, bnext = 0.0f;
      auto ask_col = [&](int c) {  // the scale and bias of chunk c (any N)
        const int n = nbase + c + (lane & 15);
        const bool in = c < cols && n < a.N;
        wnext = in ? __ldg(a.ws + n) : 0.0f;
        bnext = bias && in ? to_f32(bias[n]) : 0.0f;
      };
      if (cols > 0) tmem_ld16(acc, v);
      if (!a.vec) ask_col(0);
      else if (res) ask(0);
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {  // uniform over the warp
        const uint4 rcur[2] = {rnext[0], rnext[1]};
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          float4 f;
          f.x = __fmul_rn(static_cast<float>(static_cast<int>(v[j])), sx);
          f.y = __fmul_rn(static_cast<float>(static_cast<int>(v[j + 1])), sx);
          f.z = __fmul_rn(static_cast<float>(static_cast<int>(v[j + 2])), sx);
          f.w = __fmul_rn(static_cast<float>(static_cast<int>(v[j + 3])), sx);
          *reinterpret_cast<float4 *>(stg + lane * kEpiPitch + j) = f;
        }
        if (c + 16 < cols) tmem_ld16(acc + c + 16, v);
        const float w1c = wnext, b1c = bnext;
        if (!a.vec) ask_col(c + 16);
        else if (res) ask(c + 16);
        __syncwarp();
        if (a.vec) {  // lane: 8 columns of rows lane / 2 and lane / 2 + 16
          const int n = nbase + c + 8 * (lane & 1);
          if (n < a.N) {  // N % 8 == 0: all eight or none
            const float4 w0 = __ldg(reinterpret_cast<const float4 *>(a.ws + n));
            const float4 w1 = __ldg(reinterpret_cast<const float4 *>(a.ws + n + 4));
            const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
            T bv[8] = {};
            if (bias) {
              const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(bias + n));
              memcpy(bv, &raw, 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = (lane >> 1) + 16 * i, m = mrow + r;
              T rv[8], o[8];
              float z[8];
              memcpy(rv, &rcur[i], 16);
              const float *src = stg + r * kEpiPitch + 8 * (lane & 1);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                z[j] = __fmul_rn(src[j], w[j]);
                if (bias) z[j] += to_f32(bv[j]);
              }
              if constexpr (ACT) apply_act(z, a.act);
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = from_f32<T>(res ? z[j] + to_f32(rv[j]) : z[j]);
              uint4 raw;
              memcpy(&raw, o, 16);
              if (m < a.M) *reinterpret_cast<uint4 *>(y + static_cast<size_t>(m) * a.N + n) = raw;
            }
          }
        } else {  // any N: lane = column lane % 16 of rows lane / 16 + 2 i
          const int n = nbase + c + (lane & 15);
          const bool in = n < a.N;
          T *yp = y + static_cast<size_t>(mrow + (lane >> 4)) * a.N + n;
          const T *rp = res + static_cast<size_t>(mrow + (lane >> 4)) * a.N + n;
          const int left = in ? a.M - mrow - (lane >> 4) : 0;  // rows of this lane: 2 i < left
          constexpr int kBatch = ACT ? 4 : 16;  // (an activation's code 16 times over is too long)
#pragma unroll 1
          for (int i0 = 0; i0 < 16; i0 += kBatch) {
            float rv[kBatch], z[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
              rv[i] = res && 2 * (i0 + i) < left ? to_f32(rp[static_cast<size_t>(2 * (i0 + i)) * a.N])
                                                 : 0.0f;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              z[i] = __fmul_rn(stg[((lane >> 4) + 2 * (i0 + i)) * kEpiPitch + (lane & 15)], w1c);
              if (bias) z[i] += b1c;
            }
            if constexpr (ACT) apply_act(z, a.act);
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
              if (2 * (i0 + i) < left)
                yp[static_cast<size_t>(2 * (i0 + i)) * a.N] = from_f32<T>(res ? z[i] + rv[i] : z[i]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(L::kTmemCols)
                 : "memory");
}

// ------------------------------------------------------------------ few rows: epilogue ----
// Sums the C split-K partials of one row and finishes it; V columns per thread.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    linear_epilogue_kernel(const int32_t *__restrict__ part, int C, const LinArgs a) {
  griddep_launch();
  griddep_wait();
  const int n = (blockIdx.x * 256 + threadIdx.x) * V, m = blockIdx.y;
  if (n >= a.N) return;
  const size_t at = static_cast<size_t>(m) * a.N + n;
  const size_t cs = static_cast<size_t>(a.M) * a.N;
  int acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0;
  for (int c = 0; c < C; ++c) {
    if constexpr (V == 4) {
      const int4 p = *reinterpret_cast<const int4 *>(part + c * cs + at);
      acc[0] += p.x;
      acc[1] += p.y;
      acc[2] += p.z;
      acc[3] += p.w;
    } else {
      acc[0] += part[c * cs + at];
    }
  }
  const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.res);
  T *y = static_cast<T *>(a.y);
  const float sx = a.xs[m];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float z = __fmul_rn(__fmul_rn(static_cast<float>(acc[j]), sx), a.ws[n + j]);
    if (bias) z += to_f32(bias[n + j]);
    z = apply_act(z, a.act);
    if (res) z += to_f32(res[at + j]);
    y[at + j] = from_f32<T>(z);
  }
}

// ----------------------------------------------------------------------------- host ----
constexpr size_t kLinHeader = 256;  // the status word
constexpr int kMaxSide = 0x7fffffff - 4096;

// Weight rows per tile: the width whose last wave wastes less. A 128-wide tile moves a third
// more operand bytes per product than a 256-wide one, counted as 1/8 more time.
inline int pick_width(int M, int N) {
  const long sms = sm_count(), tm = (M + kTileM - 1) / kTileM;
  const long w256 = (tm * ((N + 255) / 256) + sms - 1) / sms;
  const long w128 = (tm * ((N + 127) / 128) + sms - 1) / sms;
  return w128 * 9 < w256 * 16 ? 128 : 256;
}

// Whether the split-K stream takes the call: at most one pass of it, and K in its 128-byte slices.
// Up to 16 rows always. Beyond, by cost in microseconds: the stream reads the weights at some 4.5
// TB/s and its partials go out and come back at 1 TB/s of their size, a tile's CTA takes 0.4 for
// each 128 columns of each K slice. Measured (stream / tiles, with residual, us): 4096 x 4096 (N x K)
// 64 rows 11.5 / 14.3, 256 rows 17.8 / 14.8; 12288 x 4096 32 rows 15.7 / 16.1, 64 rows 19.7 / 16.0; 1024 x
// 4096 256 rows 12.2 / 14.3; 151936 x 4096 8 rows 108 / 124, 64 rows 182 / 118, 256 rows 427 / 166
// (622 MB of partials). Over N of 256 to 151936, K of 1024 to 12288 and 1 to 256 rows the choice costs 0.5
// % on average and at worst 1.4 times (256 x 1024, 256 rows: 10.0 / 7.1).
inline int few_rows_limit(int M, int N, int K) {  // most rows that stream among those of M's token tiles
  if (M > 256 || K % 128 != 0) return 0;
  const int C = s8b_gemm_tc_split_count(M, N, K), NT = pick_width(M, N);
  const long sms = sm_count(), tiles = (M + kTileM - 1l) / kTileM * ((N + NT - 1l) / NT);
  const double tiled = 0.4 * (NT / 128) * (K / kSlice) * ((tiles + sms - 1) / sms);
  const double rows = (tiled - static_cast<double>(N) * K / 4.5e6) / (4.0 * C * N / 1e6);
  return rows < 16 ? 16 : rows < 256 ? static_cast<int>(rows) : 256;
}
inline bool few_rows(int M, int N, int K) {
  return M <= 16 ? K % 128 == 0 : M <= few_rows_limit(M, N, K);
}

template <typename T, int NT, bool ACT>
int launch_linear(const int8_t *xq, const int8_t *w, LinArgs a, int K, cudaStream_t st) {
  using L = LinLayout<NT, ACT>;
  CUtensorMap mx, mw;
  int rc = make_map_2d(&mx, xq, K, a.M, K, kSlice, kTileM);
  if (!rc) rc = make_map_2d(&mw, w, K, a.N, K, kSlice, NT);
  if (rc) return rc;
  a.kc = (K + kSlice - 1) / kSlice;
  a.tiles_m = (a.M + kTileM - 1) / kTileM;
  a.tiles_n = (a.N + NT - 1) / NT;
  const long tiles = static_cast<long>(a.tiles_m) * a.tiles_n;
  if (tiles > 0x7fffffffl - 4096) return S8B_ERR_SHAPE;
  auto kern = linear_tc_kernel<T, NT, ACT>;
  ensure_smem(reinterpret_cast<const void *>(kern), L::kSmem);
  const int grid = static_cast<int>(tiles < sm_count() ? tiles : sm_count());
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(L::kThreads), L::kSmem, st, mx, mw, a);
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return S8B_ERR_CUDA;
  }
  return check_launch();
}

template <typename T>
int launch_few(const int8_t *xq, const float *xs, const int8_t *w, const LinArgs &a, int K,
               void *workspace, int dtype, void *stream) {
  const int C = s8b_gemm_tc_split_count(a.M, a.N, K);
  if (C < 1) return C;
  int32_t *part = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(workspace) + kLinHeader);
  // Ordered: the caller's weights may come from a kernel just before (quantized on this stream).
  const int rc = s8b_gemm_w8a8_tc(xq, xs, w, nullptr, part, 2 | S8B_GEMM_ORDERED, a.M, a.N, K,
                                  dtype, workspace, kLinHeader, stream);
  if (rc) return rc;
  const bool v4 = a.N % 4 == 0;
  const int cols = 256 * (v4 ? 4 : 1);
  const dim3 grid((a.N + cols - 1) / cols, a.M);
  const cudaError_t e =
      v4 ? launch_pdl(linear_epilogue_kernel<T, 4>, grid, dim3(256), 0, (cudaStream_t)stream,
                      static_cast<const int32_t *>(part), C, a)
         : launch_pdl(linear_epilogue_kernel<T, 1>, grid, dim3(256), 0, (cudaStream_t)stream,
                      static_cast<const int32_t *>(part), C, a);
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return S8B_ERR_CUDA;
  }
  return check_launch();
}

}  // namespace
}  // namespace s8b

using namespace s8b;

// What a call that streams its weights needs.
static size_t stream_need(int M, int N, int K) {
  return kLinHeader + sizeof(int32_t) * s8b_gemm_tc_split_count(M, N, K) * M * N;
}

// What every call of up to M rows needs, for M <= 256.
extern "C" size_t s8b_linear_workspace_size(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > 256 || K % 128 != 0 || N > kMaxSide) return kLinHeader;
  if (M > kTileM && few_rows_limit(M, N, K) <= kTileM) M = kTileM;  // none of the second token tile
  const int most = few_rows_limit(M, N, K);
  return stream_need(M < most ? M : most, N, K);
}

extern "C" int s8b_linear_w8a8(const int8_t *xq, const float *xs, const int8_t *w,
                               const float *ws, const void *bias, int activation,
                               const void *residual, void *y, int M, int N, int K, int dtype,
                               void *workspace, size_t workspace_bytes, void *stream) {
  if (!xq || !xs || !w || !ws || !y) return S8B_ERR_ARG;
  if (activation < kActNone || activation > kActRelu) return S8B_ERR_ARG;
  if (dtype != S8B_BF16 && dtype != S8B_FP16) return S8B_ERR_DTYPE;
  // |sum| <= K * 128 * 128 stays below 2^31 for K < 2^17; rows and columns are counted in 32 bits, up
  // to a tile (or a block of the few rows' second launch) beyond the last
  if (M < 0 || N <= 0 || K <= 0 || K % 16 != 0 || K >= 131072 || M > kMaxSide || N > kMaxSide)
    return S8B_ERR_SHAPE;
  if (!aligned(xq, 16) || !aligned(w, 16) || !aligned(xs, 4) || !aligned(ws, 4) ||
      !aligned(y, 2) || !aligned(bias, 2) || !aligned(residual, 2))
    return S8B_ERR_ALIGN;
  const bool few = M > 0 && few_rows(M, N, K);
  if (!workspace || workspace_bytes < (few ? stream_need(M, N, K) : kLinHeader))
    return S8B_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return S8B_ERR_ALIGN;
  if (M == 0) return S8B_OK;
  LinArgs a = {};
  a.xs = xs;
  a.ws = ws;
  a.bias = bias;
  a.res = residual;
  a.y = y;
  a.status = static_cast<int32_t *>(workspace);
  a.M = M;
  a.N = N;
  a.act = activation;
  a.vec = N % 8 == 0 && aligned(y, 16) && aligned(bias, 16) && aligned(residual, 16) &&
          aligned(ws, 16);
  S8B_DISPATCH_DTYPE(dtype, T, {
    if (few) return launch_few<T>(xq, xs, w, a, K, workspace, dtype, stream);
    auto st = (cudaStream_t)stream;
    const bool act = activation != kActNone;
    if (pick_width(M, N) == 256)
      return act ? launch_linear<T, 256, true>(xq, w, a, K, st)
                 : launch_linear<T, 256, false>(xq, w, a, K, st);
    return act ? launch_linear<T, 128, true>(xq, w, a, K, st)
               : launch_linear<T, 128, false>(xq, w, a, K, st);
  });
  return S8B_OK;
}
