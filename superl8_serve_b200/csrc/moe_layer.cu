// A whole sparse-MoE feed-forward for up to 16 rows in one launch (s8b_moe_layer): router,
// softmax, top-k, the chosen experts' W8A8 gate_up, SwiGLU, int8 quantization, W8A8 down and
// the weighted sum.
//
// With so few rows the layer is the chosen experts' weights read once (3 H F bytes each: 38 MB
// for one row of a 2048 x 768 x 8 layer, 5.8 us at the measured copy rate), and the seven launches
// of the general path cost more than that. Here one cooperative launch of one CTA per SM runs
// three phases with a grid barrier between them:
//   A  logits: expert e's gate row against every row, all warps (float64 sums);
//   B  every CTA finds all rows' experts by itself (a warp per row, 8 rounds of a warp-wide
//      maximum), and the (chosen expert, f) pairs, gate row f and up row F + f each, are cut
//      by cost over all warps of the grid; act = silu(g) u goes to the workspace in binary32;
//   C  every CTA quantizes the act rows and computes its slice of output columns over all
//      chosen experts, so the weighted sum needs no third barrier and no atomics.
// Products are dp4a on CUDA cores: an expert has one or two rows here, where the stream of
// weights, not arithmetic, sets the time, and an MMA tile would be empty. Sums over experts are in
// ascending expert order: the result does not depend on timing.
//
// Measured (2048 x 768, 8 of 128 experts; us, in a graph / by the call, beside the bytes at the copy
// rate): one row 19.4 / 22 (6.0), eight rows 63 / 64 (37.6; 3.9 TB/s); 16 rows of 1040 x 272, 3 of
// 20, 23.6 / 25.3 (2.4). The seven launches on the same rows, with every layer's weights from HBM:
// 81, 123 and 31 beside 20, 65 and 25. The kernel spills 124 bytes a thread of its 128 registers.
// One row's time is latency: the phases wait for one another, each with its own cold loads; eight
// rows' is the stream of weights. Rings of bulk copies per warp were slower (about 125 cycles of
// issue per copy and SM), and fetching the down weights into L2 during phase B gained nothing.
//
// Numerics: logits are float64 sums rounded to binary32; integer products are exact; everything
// else is binary32, rounded to the activation dtype once, at the end. (The general path rounds
// to dtype after gate_up, silu, the product, down, the weighting and each addition.)
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace s8b {
namespace {

namespace ml {
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxT = 16, kMaxE = 256, kMaxK = 16, kMaxA = kMaxT * kMaxK;
constexpr int kMaxH = 8192;
constexpr int kCols = 8;  // columns of one expert that a warp computes together
constexpr int kSmem = 208 * 1024;  // row codes and contributions
constexpr size_t kOffBar = 64, kHeader = 256;  // workspace: status word, barrier counter
constexpr size_t kLogits = kHeader;            // fp32 [T][E]
constexpr size_t kAct = kLogits + sizeof(float) * kMaxT * kMaxE;  // fp32 [A][F]
}  // namespace ml

struct MoeArgs {
  const void *y;
  const int8_t *xq, *gu_w, *d_w;
  const float *xs, *gate, *gu_s, *d_s;
  void *out;
  uint8_t *ws;
  int T, H, F, E, k, norm;
  int code_bytes, slice;  // shared memory: row codes, then [A][slice] contributions
  float scaling;
};

// Every thread's writes before are seen by every thread of the grid after. Bounded: false after
// about a second, with the status word set. A CTA that gives up also sets the counter's top bit: the
// other CTAs, and those of every later launch, then neither wait nor go on, for the arrivals of
// a launch that gave up are not a multiple of the grid, and a barrier counted on them would open before
// all CTAs came. The caller zeroes both. (The bit comes with the arrival itself; reading the
// status word first took 0.4 us of one row's 19.4.)
constexpr unsigned long long kGaveUp = 1ull << 63;
__device__ bool grid_barrier(uint8_t *ws, int *ok) {
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long *ctr = reinterpret_cast<unsigned long long *>(ws + ml::kOffBar);
    const unsigned long long n = gridDim.x;
    __threadfence();
    const unsigned long long old = atomicAdd(ctr, 1ull), goal = (old / n + 1) * n;
    const uint32_t t0 = static_cast<uint32_t>(clock());
    bool came = (old & kGaveUp) == 0;
    while (came) {
      unsigned long long v;
      asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(ctr) : "memory");
      if (v & kGaveUp) came = false;
      else if (v >= goal) break;
      else if (static_cast<uint32_t>(clock()) - t0 > 2000000000u) {
        atomicOr(ctr, kGaveUp);
        *reinterpret_cast<volatile int32_t *>(ws) = S8B_ERR_TIMEOUT;
        came = false;
      }
    }
    *ok = came;
    __threadfence();
  }
  __syncthreads();
  return *ok != 0;
}

__device__ __forceinline__ int dot16(int4 a, int4 b, int acc) {
  acc = __dp4a(a.x, b.x, acc);
  acc = __dp4a(a.y, b.y, acc);
  acc = __dp4a(a.z, b.z, acc);
  return __dp4a(a.w, b.w, acc);
}
__device__ __forceinline__ int4 ld_stream(const int8_t *p) {  // weights: read once, not kept in L1
  int4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// What a pair of an expert with `rows` rows costs: mostly its weights, which come once, and a
// little for each row (with equal shares a CTA whose expert had 6 of 16 rows took 15,000 cycles
// where most took 6,400).
__device__ __forceinline__ int pair_cost(int rows) { return 8 + rows; }
// order of logits as unsigned integers; NaN lowest
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

// W weight rows of `bytes` bytes at w[i] against rows x[r] (shared memory, `pitch` bytes apart):
// sums[i][r] for R rows, complete in every lane. Chunks of 16 bytes, lane by lane, U at a time.
template <int W, int R, int U>
__device__ __forceinline__ void dot_rows(const int8_t *const (&w)[W], const int8_t *const (&x)[R],
                                         int bytes, int lane, int (&sums)[W][R]) {
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) sums[i][r] = 0;
  for (int c0 = 16 * lane; c0 < bytes; c0 += U * 512) {
    int4 v[W][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < W; ++i)
        v[i][u] = c0 + 512 * u < bytes ? ld_stream(w[i] + c0 + 512 * u) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + 512 * u >= bytes) break;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int4 xv = *reinterpret_cast<const int4 *>(x[r] + c0 + 512 * u);
#pragma unroll
        for (int i = 0; i < W; ++i) sums[i][r] = dot16(v[i][u], xv, sums[i][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) sums[i][r] = __reduce_add_sync(0xffffffffu, sums[i][r]);
}

// Row `warp`'s experts and weights from its logits: lane c holds experts c, c + 32, ..
template <int kC>
__device__ __forceinline__ void choose(const MoeArgs &a, const float *row, int warp, int lane,
                                       int *topi, float *topw, uint32_t *members) {
  const int E = a.E, k = a.k;
  uint32_t key[kC];
  float l[kC], m = -INFINITY;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int e = lane + 32 * c;
    l[c] = e < E ? __ldcg(row + e) : -INFINITY;
    key[c] = order_key(l[c]);
    m = fmaxf(m, l[c]);
  }
  m = warp_max_redux(m);
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < kC; ++c) s += lane + 32 * c < E ? __expf(l[c] - m) : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  uint32_t left = 0;  // this lane's experts that are still to be had
#pragma unroll
  for (int c = 0; c < kC; ++c) left |= (lane + 32 * c < E ? 1u : 0u) << c;
  int mine = 0;  // lane j keeps the j-th choice
  for (int r = 0; r < k; ++r) {  // the largest logit left, the lowest index among equals
    uint32_t bk = 0;
    int be = 0x7fffffff;
#pragma unroll
    for (int c = 0; c < kC; ++c)
      if ((left >> c & 1u) && (key[c] > bk || be == 0x7fffffff)) {
        bk = key[c];
        be = lane + 32 * c;
      }
    const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
    const int e = __reduce_min_sync(0xffffffffu, bk == best ? be : 0x7fffffff);
    if (be == e) left &= ~(1u << (e >> 5));
    if (lane == r) mine = e;
  }
  float pick = 0.0f;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const float v = __shfl_sync(0xffffffffu, l[c], mine & 31);
    if (mine >> 5 == c) pick = v;
  }
  const float p = lane < k ? __expf(pick - m) / s : 0.0f;
  float total = p;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);  // k <= 16
  if (lane < k) {
    topw[warp * k + lane] = (a.norm ? p / fmaxf(total, 1e-9f) : p) * a.scaling;
    topi[warp * k + lane] = mine;
    atomicOr(&members[mine], 1u << warp);
  }
}

template <typename T>
__global__ void __launch_bounds__(ml::kThreads, 1) moe_layer_kernel(const MoeArgs a) {
  using namespace ml;
  extern __shared__ __align__(16) int8_t rows_s[];  // x codes [T][H], later act codes [A][F]
  __shared__ float topw[kMaxA], scale_s[kMaxA];     // by assignment / by sorted row
  __shared__ int topi[kMaxA], order[kMaxA];         // expert; sorted row -> token
  __shared__ int place[kMaxA];                      // token's rows in ascending order
  __shared__ float weight[kMaxA], xs_s[kMaxT];      // and their weights; rows' scales
  __shared__ uint32_t members[kMaxE];               // rows of each expert, a bit each
  __shared__ int expert[kMaxA], offset[kMaxA + 1];  // chosen experts ascending; their first row
  __shared__ int n_experts, ok_s;
  __shared__ double part_s[kWarps][kMaxT];
  __shared__ int before[kMaxA + 1];    // cost of a pair of every chosen expert before
  __shared__ uint8_t slot_of[kMaxE];  // its place among the chosen experts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int T_ = a.T, H = a.H, F = a.F, E = a.E, k = a.k, A = T_ * k;
  float *logits = reinterpret_cast<float *>(a.ws + kLogits);
  float *act = reinterpret_cast<float *>(a.ws + kAct);
  float *contrib = reinterpret_cast<float *>(rows_s + a.code_bytes);  // [A][slice]

  // ---- A: logits ----
  for (int i = 16 * threadIdx.x; i < T_ * H; i += 16 * kThreads)
    *reinterpret_cast<int4 *>(rows_s + i) = *reinterpret_cast<const int4 *>(a.xq + i);
  // A thread keeps 8 gate values at a time (in float64 once for all rows); a row's products add
  // up over the warp's lanes, then over the warps.
  // (Few experts: several CTAs share an expert's rows.)
  const int groups = max(1, min(T_, static_cast<int>(gridDim.x) / E));
  for (int unit = blockIdx.x; unit < E * groups; unit += gridDim.x) {
    const int e = unit % E, grp = unit / E;
    const int ta = grp * T_ / groups, tb = (grp + 1) * T_ / groups;
    const float *g = a.gate + static_cast<size_t>(e) * H;
    double mine = 0.0;  // lane t: row t's sum over this warp's columns
    for (int i0 = 256 * warp; i0 < H; i0 += 256 * kWarps) {
      const int i = i0 + 8 * lane;
      double gd[8];
      float4 g0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), g1 = g0;
      if (i < H) {
        g0 = *reinterpret_cast<const float4 *>(g + i);
        g1 = *reinterpret_cast<const float4 *>(g + i + 4);
      }
      gd[0] = g0.x, gd[1] = g0.y, gd[2] = g0.z, gd[3] = g0.w;
      gd[4] = g1.x, gd[5] = g1.y, gd[6] = g1.z, gd[7] = g1.w;
#pragma unroll 4
      for (int t = ta; t < tb; ++t) {
        T v[8];
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (i < H)
          raw = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.y) +
                                                 static_cast<size_t>(t) * H + i);
        memcpy(v, &raw, 16);
        double s = 0.0;
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fma(static_cast<double>(to_f32(v[q])), gd[q], s);
        s = warp_sum_d(s);
        if (lane == t) mine += s;
      }
    }
    if (lane < T_) part_s[warp][lane] = mine;
    __syncthreads();
    if (threadIdx.x >= ta && threadIdx.x < tb) {
      double sum = 0.0;
      for (int q = 0; q < kWarps; ++q) sum += part_s[q][threadIdx.x];
      logits[threadIdx.x * E + e] = static_cast<float>(sum);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < E; i += kThreads) members[i] = 0u;
  if (threadIdx.x < T_) xs_s[threadIdx.x] = a.xs[threadIdx.x];
  if (!grid_barrier(a.ws, &ok_s)) return;

  // ---- B: each row's experts, then their gate_up and SwiGLU ----
  if (warp < T_) {
    if (E <= 128) choose<4>(a, logits + warp * E, warp, lane, topi, topw, members);
    else choose<kMaxE / 32>(a, logits + warp * E, warp, lane, topi, topw, members);
  }
  __syncthreads();
  if (warp == 0) {  // chosen experts in ascending order, and where their rows begin
    int n = 0, rows = 0, cost = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const uint32_t who = e0 + lane < E ? members[e0 + lane] : 0u;
      const uint32_t hit = __ballot_sync(0xffffffffu, who != 0u);
      // rows before, and the cost of a pair before (see pair_cost), in one scan
      const int c = __popc(who);
      uint32_t own = who ? c | static_cast<uint32_t>(pair_cost(c)) << 16 : 0u, inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (who) {
        const int at = n + __popc(hit & ((1u << lane) - 1u));
        expert[at] = e0 + lane;
        slot_of[e0 + lane] = static_cast<uint8_t>(at);
        offset[at] = rows + ((inc - own) & 0xffffu);
        before[at] = cost + ((inc - own) >> 16);
      }
      n += __popc(hit);
      const uint32_t all = __shfl_sync(0xffffffffu, inc, 31);
      rows += all & 0xffffu;
      cost += all >> 16;
    }
    if (lane == 0) {
      offset[n] = rows;
      before[n] = cost;
      n_experts = n;
    }
  }
  __syncthreads();
  const int n_ex = n_experts;
  for (int i = threadIdx.x; i < A; i += kThreads) {
    const int e = topi[i], t = i / k;
    const int p = offset[slot_of[e]] + __popc(members[e] & ((1u << t) - 1u));
    order[p] = t;
    int rank = 0;  // among the token's experts
    for (int q = 0; q < k; ++q) rank += topi[t * k + q] < e;
    place[t * k + rank] = p;
    weight[t * k + rank] = topw[i];
  }
  // this CTA's output columns
  const int h0 = static_cast<int>(static_cast<long long>(blockIdx.x) * H / gridDim.x);
  const int nh = static_cast<int>(static_cast<long long>(blockIdx.x + 1) * H / gridDim.x) - h0;
  __syncthreads();
  {
    // This warp's pairs: cost c of the whole lies in pair (c - before F) / cost of its expert;
    // lane 0 looks up where the warp's share begins, lane 1 where it ends.
    const uint32_t total = static_cast<uint32_t>(before[n_ex]) * F, nw = gridDim.x * kWarps;
    const uint32_t wg = blockIdx.x * kWarps + warp + (lane & 1);
    const uint32_t c = wg * (total / nw) + wg * (total % nw) / nw;
    int lo = 0, hi = n_ex;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<uint32_t>(before[mid]) * F <= c) lo = mid;
      else hi = mid;
    }
    const uint32_t per = before[lo + 1] - before[lo];
    const int pair =
        c >= total ? n_ex * F : lo * F + static_cast<int>((c - before[lo] * F + per - 1) / per);
    const int u1 = __shfl_sync(0xffffffffu, pair, 1);
    for (int u = __shfl_sync(0xffffffffu, pair, 0); u < u1;) {
      const int at = u / F, f = u - at * F;
      const int two = u + 1 < u1 && f + 1 < F;  // a second pair of the same expert
      const size_t base = static_cast<size_t>(expert[at]) * 2 * F;
      const int f1 = f + two;
      const int8_t *w[4] = {a.gu_w + (base + f) * H, a.gu_w + (base + F + f) * H,
                            a.gu_w + (base + f1) * H, a.gu_w + (base + F + f1) * H};
      const int lo = offset[at], hi = offset[at + 1];
      // lane 4 i + r finishes pair i, row r; its scales come with the weights
      const int i = lane >> 2 & 1, r = lane & 3;
      float sg = 0.0f, su = 0.0f;
      if (lane < 8) {
        sg = a.gu_s[base + (i ? f1 : f)];
        su = a.gu_s[base + F + (i ? f1 : f)];
      }
      auto rows = [&](auto n, int p0) {  // n of the expert's rows, from p0 on
        constexpr int R = decltype(n)::value;
        const int8_t *x[R];
#pragma unroll
        for (int q = 0; q < R; ++q) x[q] = rows_s + order[min(p0 + q, hi - 1)] * H;
        int sum[4][R];
        dot_rows<4, R, 4>(w, x, H, lane, sum);
        int gs = 0, us = 0;
#pragma unroll
        for (int q = 0; q < R; ++q)
          if (q == r) {
            gs = i ? sum[2][q] : sum[0][q];
            us = i ? sum[3][q] : sum[1][q];
          }
        if (r < R && p0 + r < hi && lane < 8 && (i == 0 || two)) {
          const float sx = xs_s[order[p0 + r]];
          const float g = static_cast<float>(gs) * sx * sg;
          const float v = static_cast<float>(us) * sx * su;
          act[static_cast<size_t>(p0 + r) * F + f + i] = g / (1.0f + __expf(-g)) * v;
        }
      };
      if (hi - lo == 1) rows(std::integral_constant<int, 1>{}, lo);
      else if (hi - lo == 2) rows(std::integral_constant<int, 2>{}, lo);
      else
        for (int p0 = lo; p0 < hi; p0 += 4) rows(std::integral_constant<int, 4>{}, p0);
      u += 1 + two;
    }
  }
  if (!grid_barrier(a.ws, &ok_s)) return;

  // ---- C: act codes, then this CTA's columns of the down products ----
  if (nh == 0) return;
  for (int p0 = warp; p0 < A; p0 += 2 * kWarps) {  // two rows at a time
    constexpr int kHold = 8;  // vectors of a row that stay in registers (1024 values)
    float4 v[2][kHold];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < kHold; ++u) {
        const int p = p0 + h * kWarps, i = 4 * lane + 128 * u;
        v[h][u] = p < A && i < F
                      ? __ldcg(reinterpret_cast<const float4 *>(act + static_cast<size_t>(p) * F + i))
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    auto top = [](float4 x) {
      return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = p0 + h * kWarps;
      if (p >= A) break;
      const float *src = act + static_cast<size_t>(p) * F;
      float mx = 0.0f;
#pragma unroll
      for (int u = 0; u < kHold; ++u) mx = fmaxf(mx, top(v[h][u]));
      for (int i = 4 * lane + 128 * kHold; i < F; i += 128)
        mx = fmaxf(mx, top(__ldcg(reinterpret_cast<const float4 *>(src + i))));
      const QParams q = qparams(warp_max_redux(mx), 127.0f);
      auto put = [&](int i, float4 x) {
        char4 c;
        c.x = static_cast<signed char>(qcode(x.x, q.inv, 127));
        c.y = static_cast<signed char>(qcode(x.y, q.inv, 127));
        c.z = static_cast<signed char>(qcode(x.z, q.inv, 127));
        c.w = static_cast<signed char>(qcode(x.w, q.inv, 127));
        *reinterpret_cast<char4 *>(rows_s + static_cast<size_t>(p) * F + i) = c;
      };
#pragma unroll
      for (int u = 0; u < kHold; ++u)
        if (4 * lane + 128 * u < F) put(4 * lane + 128 * u, v[h][u]);
      for (int i = 4 * lane + 128 * kHold; i < F; i += 128)
        put(i, __ldcg(reinterpret_cast<const float4 *>(src + i)));
      if (lane == 0) scale_s[p] = q.scale;
    }
  }
  __syncthreads();
  {
    // eight columns of one expert at a time: they come from L2, whose latency needs the loads
    const int per = (nh + kCols - 1) / kCols, units = n_ex * per;
    for (int u = warp; u < units; u += kWarps) {
      const int at = u / per, c0 = kCols * (u - at * per);
      const size_t row = static_cast<size_t>(expert[at]) * H + h0;
      const int8_t *w[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) w[i] = a.d_w + (row + min(c0 + i, nh - 1)) * F;
      const int i = lane >> 2, r = lane & 3;  // lane 4 i + r finishes column i, row r
      const float sd = c0 + i < nh ? a.d_s[row + c0 + i] : 0.0f;
      const int lo = offset[at], hi = offset[at + 1];
      auto rows = [&](auto n, int p0) {
        constexpr int R = decltype(n)::value;
        const int8_t *x[R];
#pragma unroll
        for (int q = 0; q < R; ++q) x[q] = rows_s + static_cast<size_t>(min(p0 + q, hi - 1)) * F;
        int sum[kCols][R];
        dot_rows<kCols, R, 2>(w, x, F, lane, sum);
        int v = 0;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int q = 0; q < R; ++q)
            if (c == i && q == r) v = sum[c][q];
        if (r < R && p0 + r < hi && c0 + i < nh)
          contrib[(p0 + r) * a.slice + c0 + i] = static_cast<float>(v) * scale_s[p0 + r] * sd;
      };
      if (hi - lo == 1) rows(std::integral_constant<int, 1>{}, lo);
      else if (hi - lo == 2) rows(std::integral_constant<int, 2>{}, lo);
      else
        for (int p0 = lo; p0 < hi; p0 += 4) rows(std::integral_constant<int, 4>{}, p0);
    }
  }
  __syncthreads();
  // a token's rows in ascending order, that is of their experts
  T *out = static_cast<T *>(a.out);
  for (int i = threadIdx.x; i < T_ * nh; i += kThreads) {
    const int t = i / nh, c = i - t * nh;
    float s = 0.0f;
    for (int j = 0; j < k; ++j) s = fmaf(weight[t * k + j], contrib[place[t * k + j] * a.slice + c], s);
    out[static_cast<size_t>(t) * H + h0 + c] = from_f32<T>(s);
  }
}

}  // namespace
}  // namespace s8b

using namespace s8b;

extern "C" size_t s8b_moe_layer_workspace_size(int top_k, int F) {
  if (top_k <= 0 || top_k > ml::kMaxK || F <= 0) return ml::kAct;
  return ml::kAct + sizeof(float) * ml::kMaxT * static_cast<size_t>(top_k) * F;
}

extern "C" int s8b_moe_layer_max_rows(int H, int F, int top_k) {
  using namespace ml;
  if (H <= 0 || F <= 0 || top_k <= 0 || top_k > kMaxK || H % 16 || F % 16 || H > kMaxH) return 0;
  const long long row = H > static_cast<long long>(top_k) * F ? H : static_cast<long long>(top_k) * F;
  const long long per = row + 4ll * top_k * ((H + 127) / 128);  // its codes, and contributions
  const long long n = (kSmem - 256) / per;                      // (a CTA's columns: fewer)
  return static_cast<int>(n < kMaxT ? n : kMaxT);
}

extern "C" int s8b_moe_layer(const void *y, const int8_t *xq, const float *xs, const float *gate,
                             const int8_t *gu_w, const float *gu_s, const int8_t *d_w,
                             const float *d_s, void *out, int T_, int H, int F, int E, int top_k,
                             int norm_topk_prob, float routed_scaling, void *workspace,
                             size_t workspace_bytes, int dtype, void *stream) {
  using namespace ml;
  if (!y || !xq || !xs || !gate || !gu_w || !gu_s || !d_w || !d_s || !out) return S8B_ERR_ARG;
  if (dtype != S8B_BF16 && dtype != S8B_FP16) return S8B_ERR_DTYPE;
  if (T_ < 0 || E <= 0 || E > kMaxE || top_k <= 0 || top_k > E ||
      T_ > s8b_moe_layer_max_rows(H, F, top_k) ||
      // pairs' costs in 32 bits: at most 24 for each of top_k T experts' F pairs
      static_cast<long long>(F) * top_k * T_ * 24 >= (1ll << 31))
    return S8B_ERR_SHAPE;
  if (!aligned(y, 16) || !aligned(xq, 16) || !aligned(gate, 16) || !aligned(gu_w, 16) ||
      !aligned(d_w, 16) || !aligned(xs, 4) || !aligned(gu_s, 4) || !aligned(d_s, 4) ||
      !aligned(out, 2))
    return S8B_ERR_ALIGN;
  if (!workspace || workspace_bytes < s8b_moe_layer_workspace_size(top_k, F))
    return S8B_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return S8B_ERR_ALIGN;
  if (T_ == 0) return S8B_OK;
  const int sms = tc::sm_count();
  MoeArgs a = {};
  a.y = y;
  a.xq = xq;
  a.xs = xs;
  a.gate = gate;
  a.gu_w = gu_w;
  a.gu_s = gu_s;
  a.d_w = d_w;
  a.d_s = d_s;
  a.out = out;
  a.ws = static_cast<uint8_t *>(workspace);
  a.T = T_;
  a.H = H;
  a.F = F;
  a.E = E;
  a.k = top_k;
  a.norm = norm_topk_prob;
  a.scaling = routed_scaling;
  const size_t row = H > top_k * F ? H : static_cast<size_t>(top_k) * F;
  a.code_bytes = static_cast<int>((row * T_ + 15) / 16 * 16);
  a.slice = (H + sms - 1) / sms;
  const size_t smem = a.code_bytes + sizeof(float) * T_ * top_k * static_cast<size_t>(a.slice);
  if (smem > kSmem) return S8B_ERR_SHAPE;
  S8B_DISPATCH_DTYPE(dtype, TT, {
    ensure_smem(reinterpret_cast<const void *>(moe_layer_kernel<TT>), smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr;  // the CTAs wait for one another: all must be resident
    attr.id = cudaLaunchAttributeCooperative;
    attr.val.cooperative = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, moe_layer_kernel<TT>, a);
    if (e != cudaSuccess) {
      record_cuda_error(e);
      return S8B_ERR_CUDA;
    }
  });
  return check_launch();
}
