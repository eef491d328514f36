// Attention of a chunk of new tokens per sequence over the paged int8 KV cache
// (s8b_paged_chunk_q8).
//
// Sequence s brings n new rows (cu_q[s] .. cu_q[s+1]) at the end of a context of c keys; row i
// sees keys 0 .. c - n + i. With int8 queries, keys and values,
//   x_j = (q . k_j) ks_j,   t_j = qs scale x_j,   o = sum_j e^(t_j - m) vs_j v_j / sum_j e^(t_j - m)
// q . k is exact (kind::i8, int32); the softmax is binary32; the products w_j = e^(..) vs_j go
// into the second product (kind::f16 with binary32 sums) as the sum of two bf16 numbers, p and
// what rounding to p left over (2^-16 of w_j at most in all), and that product runs once for
// each; its other operand, the value codes, bf16 holds exactly. bf16 rather than fp16: its
// range is binary32's, so no token's scale can overflow or vanish beside another's. One term alone
// (2^-8 at most) shows beside the output's own rounding: the root of the mean square error
// against 64 bits was 2.3e-3 for bf16 results (2.8e-3 behind 37 keys) where that rounding makes
// 1.7e-3, and 1.7e-3 for fp16 results where it makes 2.1e-4. The second term costs 3
// to 8 % (by the call: eight prompts of up to 2048 rows 354 -> 382 us, 64 sequences of up to 4
// draft rows 82 -> 86, 5 rows over 37 keys nothing).
//
// Bound. Each score (row x key) costs 2 x 128 int8 and 2 x 128 bf16 operations, one exponential
// and about 5 further instructions; a key's bytes serve 128 rows. Above some 16 rows per sequence
// the products set the floor (1635 TFLOP/s measured for bf16, twice that counted for int8), below it
// the keys' 264 bytes per head. What bounds the kernel is the chain from S to P: a step of 64 keys
// took a softmax group 850 cycles alone, 1270 beside the other group and about 1900 beside the
// converters too, against 512 of tensor work for both groups; with few rows the conversion of V,
// 2000 of the 2500 cycles of a tile of 128 keys (counted with one weight term; with two, the issue
// slots are 46 % and the tensor pipe 31 % busy over eight prompts). The kernel has 128 registers a
// thread at its launch, shared out as 176 and 80, and spills 28 bytes.
//
// Measured (us, in a graph / by the call, beside the floor): 4096 new rows over 16K keys, 32 heads
// on 4, fp16, 1312 / 1375 (442); eight prompts of up to 2048 rows, 32 on 8, 376 / 382 (77), where the
// row-by-row prefill attention takes 8673; 64 sequences x up to 4 draft rows over up to 2048 keys 87 /
// 87 (27 at the copy rate; 156); 2 sequences x 16 rows over 64K keys, 40 on 8, 73 / 72 (21); 5 rows
// over 37 keys 15 / 18 (14).
//
// Unit of work. The G query heads of a kv head share its keys, so a tile's 128 rows are
// 128 / G tokens x G heads, and an item is two such tiles (A and B) of one sequence and kv head:
// each K/V tile of 128 keys is staged and converted once for both, and while the softmax of
// one tile runs, the tensor pipe works for the other. All items' key tiles in a row are cut
// into equal runs, one per CTA, whatever the lengths: a CTA takes several items, or many CTAs
// one item's keys. An item that a cut splits leaves partials (o, m, l) in the workspace, which
// chunk_merge_kernel joins in key order, so the result does not depend on timing.
//
// Roles (16 warps): 0-3 and 4-7 softmax of groups A and B; 8-11 convert V codes to bf16; 12 and
// 13 issue the MMAs of A and B (one warp for both was the bottleneck: a wait that is already
// satisfied takes 110 cycles and more, and each tile needs four); 14 walks the work list and
// loads K pages and scales, 15 loads Q and V pages. Items of one tile of rows (few new tokens)
// give group B the odd key tiles of the same rows.
// TMEM: S_A | S_B | O_A | O_B, 128 columns each; the weights P overwrite the S they came from.
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace s8b {
namespace {

using namespace tc;

namespace ca {
constexpr int kHd = 128;
constexpr int kThreads = 512;
constexpr int kKeys = 128;        // keys per tile
constexpr int kRows = 128;        // rows per tile
constexpr int kStages = 3;
// Barriers that tell of a stage's K. A parity tells only one phase from the next, so a wait for
// tile j is right only if the barrier's last use before is known to have landed, and none after j
// can. Where the groups share a piece's key tiles, a group waits for every second tile alone: with a
// barrier per stage the use before tile j is tile j - 3, which the other group waited for. Six
// barriers keep the groups apart: the use before is tile j - 6, the group's own (or of an
// earlier piece, all of whose K has landed when the next piece's queries come), and the use
// after waits for this group's reads of tile j.
constexpr int kFull = 2 * kStages;
constexpr int kTile = kKeys * kHd;                 // one int8 tile (16 KB)
constexpr int kStage = 2 * kTile + 2 * kKeys * 4;  // K | V | ks | vs
constexpr int kOffVs = kStages * kStage;           // V in bf16: 2 buffers of 2 panels of 64 dims
constexpr int kV16 = 2 * kTile;
constexpr int kOffQ = kOffVs + 2 * kV16;           // Q tiles A, B
constexpr int kOffBar = kOffQ + 2 * kTile;
constexpr int kPieces = 4;        // pieces announced ahead
constexpr int kOffSums = kOffBar + 1024;
constexpr int kOffSeq = kOffSums + 1024;             // prefix[S+1] int64, cu[S+1], ctx[S]
constexpr int kMaxSeqs = 1024;
constexpr int kSeqBytes = (kMaxSeqs + 1) * 8 + (kMaxSeqs + 1) * 4 + kMaxSeqs * 4;
constexpr int kSmem = 1024 + kOffSeq + kSeqBytes;
constexpr int kItemRows = 2 * kRows;
// What an item costs beside its key tiles (queries, the softmax's start, its result), in tiles:
// it counts so many units more, before its first key tile. Times (us) with 0, 1, 3 and 5 units: eight
// prompts of up to 2048 rows 406, 381, 376, 395; 32 of up to 700 rows 300, 282, 279, 278; 64 sequences of
// 4 draft rows over 2K keys 92, 90, 87, 86; 24 of 16 rows over 4K keys 72, 67, 66, 66; 2 x 16 rows over
// 64K keys 77, 75, 73, 73; 500 rows over 30K keys 761, 756, 757, 759.
constexpr int kItemUnits = 3;
constexpr float kSumMax = 0x1p60f;  // a tile's sum of e^(t - reference) above: a new reference
constexpr int kMaxCtas = 512;     // CTAs the workspace has room for
// workspace: status word, per-CTA metadata, partials
struct Meta {  // an item whose first piece is CTA c's (slot 2c + 1); pieces go on in slots 2c' + 0
  int valid, t0, ntok, g, last;
  int pad[3];
};
constexpr size_t kOffMeta = 256;
constexpr size_t kOffMl = kOffMeta + sizeof(Meta) * kMaxCtas;
constexpr size_t slot_ml = kItemRows * 2, slot_o = kItemRows * kHd;
}  // namespace ca

struct ChunkArgs {
  const int8_t *q;
  const float *qs;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *bt, *ctx, *cu;
  void *out;
  uint8_t *ws;
  float *ml, *po;
  int T, S, Hq, Hkv, G, TA, TN, bs_log2, max_blocks, num_blocks;
  int cap;     // positions that a block-table row reaches
  int copies;  // pages go by bulk copies
  float c;     // scale * log2(e)
};

// ------------------------------------------------------------------- small PTX pieces ----
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
        "l"(reinterpret_cast<unsigned long long &>(c)));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float2 v) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
  return r;
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
        "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_16x256_x1(uint32_t addr, uint32_t *v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_16x256_x4(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,"
      "%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_16x256_x1(uint32_t addr, const uint32_t *v) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x1.b32 [%4], {%0,%1,%2,%3};" ::"r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(addr));
}
__device__ __forceinline__ void tmem_st_16x128_x8(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,"
      "%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(addr));
}
__device__ __forceinline__ void tmem_ld_16x256_x2(uint32_t addr, uint32_t *v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// What packing v to two bf16 left over, packed: exact differences, rounded again.
__device__ __forceinline__ uint32_t pack_rest(float2 v, uint32_t p) {
  return pack_bf16(add2(v, make_float2(-__uint_as_float(p << 16), -__uint_as_float(p & 0xffff0000u))));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives on `bar` when all of this thread's cp.async so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// All of this thread's cp.async have landed.
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Bounded wait, about a second. Short on purpose: instruction fetch bounds this kernel's
// single-thread roles, because all roles' code competes for the SM's instruction caches (with
// longer waits and every loop unrolled, 200 KB of it, a wait already satisfied took 350 cycles).
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *abort,
                                         int32_t *status) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = static_cast<uint32_t>(clock());
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*abort) return false;
    if (static_cast<uint32_t>(clock()) - t0 > 2000000000u) {
      *abort = 1;
      *reinterpret_cast<volatile int32_t *>(status) = S8B_ERR_TIMEOUT;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int c0, int c1, int c2,
                                            uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t *bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n)
               : "memory");
}
// D[128 x 128] (+)= A (bf16 in TMEM, 8 columns per 16 keys) . B (shared memory)
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(z), "r"(z), "r"(z), "r"(z));
}
// kind::f16: D f32 (1) at bit 4, A and B bf16 (1) at 7 and 10, B MN-major at 16, N, M.
constexpr uint32_t kIdescPv =
    (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
// B operand V [keys][dims], dims contiguous, two panels of 64 dims: 8-key groups 1024 B apart
// (stride), panels 16 KB apart (leading).
__device__ __forceinline__ uint64_t v16_desc(uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(16384 >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// Two int8 codes in the low bytes of x's halves -> two bf16: a code c is (c & 127) minus 128 if
// its sign bit is set; 128 + (c & 127) and 128 (or 256) are bf16 numbers made by their bits,
// and their difference is exact.
__device__ __forceinline__ uint32_t codes_bf16(uint32_t x) {
  const uint32_t a = (x & 0x007F007Fu) | 0x43004300u, b = (x & 0x00800080u) | 0x43004300u;
  __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(a),
                             reinterpret_cast<const __nv_bfloat162 &>(b));
  return reinterpret_cast<uint32_t &>(r);
}

// ---------------------------------------------------------------------- the work list ----
// Item (sequence, kv head, tile of 2 TA tokens). units = kItemUnits and its key tiles, at least
// one. A cut among an item's first units is moved to its start, so that no piece is without keys.
struct SeqTab {
  const long long *pre;  // [S + 1] units before each sequence
  const int *cu, *ctx;
};
struct Item {
  int t0, ntok, base, keys, nk, units;  // first row, tokens, keys before row t0, keys, tiles
};
__device__ __forceinline__ Item item_at(const SeqTab &q, const ChunkArgs &a, int s, int t) {
  Item it;
  const int c0 = q.cu[s], n = q.cu[s + 1] - c0, i0 = t * 2 * a.TA;
  const int cap = a.cap;
  it.t0 = c0 + i0;
  it.ntok = min(2 * a.TA, n - i0);
  it.base = q.ctx[s] - n + i0;
  it.keys = min(max(it.base + it.ntok, 0), cap);
  it.nk = (it.keys + ca::kKeys - 1) / ca::kKeys;
  it.units = ca::kItemUnits + max(it.nk, 1);
  return it;
}
// Row rr of a 128-row tile -> its token (of the tile) and head (of the kv head's); false: none.
// Usually token by token. An item of up to 32 / G tokens is narrow: each softmax warp gets up to
// 8 rows of it, its first ones, a quarter of a warp's work (see the softmax).
__device__ __forceinline__ bool place(const ChunkArgs &a, int ntok, int rr, int *tok, int *head) {
  const bool narrow = ntok <= 4 * a.TN;
  const int i = narrow ? rr & 31 : rr, t = i / a.G;
  *head = i - t * a.G;
  *tok = narrow ? (rr >> 5) * a.TN + t : t;
  return t < (narrow ? a.TN : a.TA);
}
// Tiles of sequence s (none if it brings no row, or its range is no range).
__device__ __forceinline__ int tiles_of(const SeqTab &q, const ChunkArgs &a, int s) {
  const int n = q.cu[s + 1] - q.cu[s];
  return n <= 0 ? 0 : n <= 2 * a.TA ? 1 : (n + 2 * a.TA - 1) / (2 * a.TA);
}
// One piece of a CTA's run: key tiles [k0, k1) of one item. Warp 14 walks the run and announces
// the pieces to the other roles through a small ring in shared memory (a walk in every role's
// registers made the softmax spill).
struct Piece {
  int valid;  // 0: the run is over
  int s, g, t0, ntok, base, keys, k0, k1;
  int starts, ends;  // holds the item's first / last key tile
  int behind;        // units of the item after this piece
};
struct Walk {
  int s, g, t, off, left;
  __device__ __forceinline__ void next(const SeqTab &q, const ChunkArgs &a, Piece *p) {
    p->valid = left > 0;
    if (left <= 0) return;
    const Item it = item_at(q, a, s, t);
    const int take = min(left, it.units - off);
    p->s = s;
    p->g = g;
    p->t0 = it.t0;
    p->ntok = it.ntok;
    p->base = it.base;
    p->keys = it.keys;
    p->k0 = max(off - ca::kItemUnits, 0);
    p->k1 = min(off + take - ca::kItemUnits, it.nk);
    p->starts = off == 0;
    p->ends = off + take == it.units;
    p->behind = it.units - (off + take);
    left -= take;
    off = 0;  // only the run's first piece starts inside an item, only its last ends there
    const int n = q.cu[s + 1] - q.cu[s];
    if (++t * 2 * a.TA < n) return;
    t = 0;
    if (++g < a.Hkv) return;
    g = 0;
    do ++s;
    while (s < a.S && q.cu[s + 1] <= q.cu[s]);
  }
};

template <typename T>
__global__ void __launch_bounds__(ca::kThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_qn, const ChunkArgs a) {
  using namespace ca;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(sm + kOffBar);  // [6] K and scales loaded
  uint64_t *vland = full + kFull;     // [3] V codes loaded
  uint64_t *empty = vland + kStages;  // [3] K read, V converted, scales read by both softmax groups
  uint64_t *vfull = empty + kStages;   // [2] bf16 V written
  uint64_t *vempty = vfull + 2;  // [2] bf16 V read
  uint64_t *sfull = vempty + 2;  // [group][half tile] S ready
  uint64_t *pfull = sfull + 4;   // [group][half tile] P written (S read, O rescaled)
  uint64_t *pvin = pfull + 4;    // [group][half tile] P V is in O
  uint64_t *ofull = pvin + 4;    // [2] a piece's O complete
  uint64_t *bdone = ofull + 2;   // group B left its sums for A (split pieces)
  uint64_t *btaken = bdone + 1;  // A has read B's O
  uint64_t *afull = btaken + 1;        // [4] piece announced
  uint64_t *aempty = afull + kPieces;  // [4] piece done by every other role's warp
  uint64_t *qfull = aempty + kPieces, *qempty = qfull + 1, *drained = qempty + 1;
  uint64_t *pdone = drained + 2;  // a piece's products done by both groups
  uint32_t *tmem_base = reinterpret_cast<uint32_t *>(pdone + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_base + 1);
  int *first = reinterpret_cast<int *>(tmem_base + 2);  // s, g, t, off of this CTA's run
  long long *run = reinterpret_cast<long long *>(sm + kOffBar + 448);  // its units: begin, end
  int *in_seq = reinterpret_cast<int *>(run + 2);                       // their sequences
  Piece *pieces = reinterpret_cast<Piece *>(sm + kOffBar + 512);
  static_assert(kPieces * sizeof(Piece) <= 512, "the ring of pieces fits its 512 bytes");
  float *bsum = reinterpret_cast<float *>(sm + kOffSums);  // [128] reference, sum of B's rows
  long long *pre = reinterpret_cast<long long *>(sm + kOffSeq);
  int *cu = reinterpret_cast<int *>(pre + kMaxSeqs + 1);
  int *ctx = cu + kMaxSeqs + 1;
  int32_t *status = reinterpret_cast<int32_t *>(a.ws);
  Meta *meta = reinterpret_cast<Meta *>(a.ws + kOffMeta);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  griddep_launch();
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kFull; ++i) mbar_init(&full[i], a.copies ? 1 + 32 : 32);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&vland[i], a.copies ? 1 : 32);
      mbar_init(&empty[i], 2 + 4 + 4 + 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&vfull[i], 4);
      mbar_init(&vempty[i], 2);
      mbar_init(&ofull[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 2);
      mbar_init(&pfull[i], 4);
      mbar_init(&pvin[i], 1);
    }
    mbar_init(bdone, 4);
    mbar_init(btaken, 4);
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&afull[i], 1);
      mbar_init(&aempty[i], 15);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, 2);
    mbar_init(pdone, 2);
    mbar_init(&drained[0], 1);
    mbar_init(&drained[1], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  griddep_wait();

  // ---- this CTA's run of units ----
  const int S = a.S;
#pragma unroll 1
  for (int i = threadIdx.x; i <= S; i += kThreads) {
    const int v = a.cu[i];
    // rows outside the tensors, or lengths that fall: cut to what exists, and said so
    if (v < 0 || v > a.T || (i > 0 && v < a.cu[i - 1])) *status = S8B_ERR_ARG;
    cu[i] = min(max(v, 0), a.T);
    if (i < S) {
      const int c = a.ctx[i];
      if (c < 0 || static_cast<long long>(c) > (static_cast<long long>(a.max_blocks) << a.bs_log2))
        *status = S8B_ERR_ARG;
      ctx[i] = max(c, 0);
    }
  }
  __syncthreads();
  const SeqTab tab{pre, cu, ctx};
  // units of each sequence: a thread adds up few tiles, a warp many
  constexpr int kFewTiles = 4;
#pragma unroll 1
  for (int s = threadIdx.x; s < S; s += kThreads) {
    const int nt = tiles_of(tab, a, s);
    if (nt > kFewTiles) continue;
    long long w = 0;
#pragma unroll 1
    for (int t = 0; t < nt; ++t) w += item_at(tab, a, s, t).units;
    pre[s + 1] = w * a.Hkv;
  }
#pragma unroll 1
  for (int s = warp; s < S; s += kThreads / 32) {
    const int nt = tiles_of(tab, a, s);
    if (nt <= kFewTiles) continue;
    long long w = 0;
#pragma unroll 1
    for (int t = lane; t < nt; t += 32) w += item_at(tab, a, s, t).units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) pre[s + 1] = w * a.Hkv;
  }
  __syncthreads();
  if (warp == 0) {
    long long carry = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < S; s0 += 32) {
      long long v = s0 + lane < S ? pre[s0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      v += carry;
      if (s0 + lane < S) pre[s0 + lane + 1] = v;
      carry = __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  __syncthreads();
  const long long W = pre[S];
  const long long ctas = min(static_cast<long long>(gridDim.x), W);  // CTAs with work
  const long long u0 = blockIdx.x < ctas ? blockIdx.x * W / ctas : 0;
  const long long u1 = blockIdx.x < ctas ? (blockIdx.x + 1) * W / ctas : 0;
  if (threadIdx.x < 2) run[threadIdx.x] = threadIdx.x ? u1 : u0;
#pragma unroll 1
  for (int s = threadIdx.x; s < S; s += kThreads) {
    if (pre[s] <= u0 && u0 < pre[s + 1]) in_seq[0] = s;
    if (pre[s] <= u1 && u1 < pre[s + 1]) in_seq[1] = s;
  }
  __syncthreads();
  // Warp 0 finds the item of unit u0, warp 1 that of u1 (none behind the last unit).
  if (warp < 2 && u1 > u0 && (warp ? u1 : u0) < W) {
    const long long u = warp ? u1 : u0;
    const int s = in_seq[warp];
    const long long per = (pre[s + 1] - pre[s]) / a.Hkv, rem = u - pre[s];
    const int g = static_cast<int>(rem / per);
    long long r = rem - g * per;  // units of this head before u
    int t0 = 0;
    const int nt = tiles_of(tab, a, s);
    while (true) {
      const int n = t0 + lane < nt ? item_at(tab, a, s, t0 + lane).units : 0;
      long long v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, v > r);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          int off = static_cast<int>(r - (v - n));
          if (off <= kItemUnits) {
            run[warp] = u - off;
            off = 0;
          }
          if (warp == 0) {
            first[0] = s;
            first[1] = g;
            first[2] = t0 + lane;
            first[3] = off;
          }
        }
        break;
      }
      r -= __shfl_sync(0xffffffffu, v, 31);
      t0 += 32;
      if (t0 >= nt) break;  // not reached: the units of the sequence hold u
    }
  }
  if (threadIdx.x == 0) meta[blockIdx.x].valid = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base;
  // Every role goes through the same pieces; `kt` counts the key tiles so far (stage kt % 3, bf16
  // V buffer kt % 2), `np` the pieces with keys. A piece is next()ed by all lanes of a warp.
  int na = 0;
  auto next = [&]() -> const Piece * {
    const bool got = bar_wait(&afull[na % kPieces], (na / kPieces) & 1, abort_flag, status);
    if (!__all_sync(0xffffffffu, got)) return nullptr;
    const Piece *p = &pieces[na % kPieces];
    return p->valid ? p : nullptr;
  };
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&aempty[na % kPieces]);
    ++na;
  };
  if (warp < 8) {
    // ------------------------------------------------------------------------ softmax ----
    // S comes in the 16x256b shape: lane l holds keys 2 (l % 4), + 1 of each group of 8 for the
    // rows l / 4 + 8 j (j = 0..3) of its warp's 32, so that a scale read from shared memory
    // serves four rows (with a row per lane the broadcast reads alone took as long as the
    // exponentials: 512 bytes of register writes for 4 values).
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(176));
    const int hf = warp >> 2, quad = lane & 3;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + hf * 128 + lanes, to = tmem + 256 + hf * 128 + lanes;
    constexpr uint32_t kLow = 16u << 16;  // rows 16..31 of the warp
    int kt = 0, ns = 0, np = 0, nsp = 0;  // tiles, this group's tiles, its pieces, split pieces
    bool ok = true;
    auto wait = [&](uint64_t *bar, int par) {
      ok = bar_wait(bar, par, abort_flag, status);
      return ok = __all_sync(0xffffffffu, ok);
    };
    while (const Piece *pc = next()) {
      const bool split = pc->ntok <= a.TA;  // one tile of rows: the groups share its key tiles
      const int tok0 = split ? 0 : hf * a.TA;
      const bool narrow = pc->ntok <= 4 * a.TN;
      auto q_row = [&](int tok, int head) {
        return static_cast<size_t>(pc->t0 + tok0 + tok) * a.Hq + pc->g * a.G + head;
      };
      float c[4], mr[4], l[4];  // log2(e) scale q_s, reference (a power of 2), sum of own keys
      int lim[4];               // keys the row sees (rows of no token: all, they mask no tile)
      int least = pc->keys;
      bool rows = false;        // the warp has rows to answer for
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int rr = 32 * (warp & 3) + (lane >> 2) + 8 * j;
        int tok, head;
        const bool valid = place(a, pc->ntok, rr, &tok, &head) && tok0 + tok < pc->ntok;
        c[j] = valid ? a.qs[q_row(tok, head)] * a.c : 0.0f;
        lim[j] = valid ? min(max(pc->base + tok0 + tok + 1, 0), pc->keys) : pc->keys;
        mr[j] = -INFINITY;
        l[j] = 0.0f;
        least = min(least, lim[j]);
        rows = rows || valid;
      }
      rows = __any_sync(0xffffffffu, rows);
      const int whole_tiles = __reduce_min_sync(0xffffffffu, least) / kKeys;
      const int k0 = pc->k0, k1 = pc->k1;
      bool fresh = true;  // O holds nothing yet
      const int step = split ? 2 : 1;
      for (int k = k0 + (split ? hf : 0); ok && k < k1; k += step) {
        const int st = (kt + k - k0) % kStages;
        const int par = ns & 1;
        ++ns;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (!wait(&sfull[2 * hf + h], par)) break;
          tc_fence_after();
          const uint32_t tu = ts + 64 * h;
          const int key0 = k * kKeys + 64 * h + 2 * quad;  // this lane's first key
          // its keys' scales: float2 index 4 * group of 8 + quad
          const float2 *ks =
              reinterpret_cast<const float2 *>(sm + st * kStage + 2 * kTile) + 32 * h + quad;
          const float2 *vs = ks + kKeys / 2;
          // One pass with the reference at hand: binary32 and bf16 keep their precision at any
          // magnitude, so the reference has to be near the row's maximum, not at it, and the sum
          // of these keys alone shows whether it still is. Returns whether it was (else nothing
          // has been written).
          auto put = [&](const uint32_t (&pk)[2][16], const uint32_t (&pl)[2][16], auto low) {
            tmem_st_16x128_x8(tu, pk[0]);
            if constexpr (decltype(low)::value) tmem_st_16x128_x8(tu + kLow, pk[1]);
            tmem_st_16x128_x8(tu + 32, pl[0]);
            if constexpr (decltype(low)::value) tmem_st_16x128_x8(tu + 32 + kLow, pl[1]);
          };
          auto pass = [&](auto masked, auto all) -> bool {
            constexpr bool kAll = decltype(all)::value;
            constexpr int J = kAll ? 4 : 1;  // rows of a lane (narrow: the warp's first 8 rows)
            float2 sum[J];
#pragma unroll
            for (int j = 0; j < J; ++j) sum[j] = make_float2(0.0f, 0.0f);
            uint32_t v[2][2][16], pk[2][16] = {}, pl[2][16] = {};
            tmem_ld_16x256_x4(tu, v[0][0]);
            if constexpr (kAll) tmem_ld_16x256_x4(tu + kLow, v[0][1]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              tmem_wait_ld();
              if (b == 0) {
                tmem_ld_16x256_x4(tu + 32, v[1][0]);
                if constexpr (kAll) tmem_ld_16x256_x4(tu + kLow + 32, v[1][1]);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float2 kf = ks[16 * b + 4 * q], vf = vs[16 * b + 4 * q];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                  const int *s = reinterpret_cast<const int *>(v[b][j >> 1]) + 4 * q + 2 * (j & 1);
                  const float2 x =
                      mul2(make_float2(static_cast<float>(s[0]), static_cast<float>(s[1])), kf);
                  const float2 t = fma2(x, make_float2(c[j], c[j]), make_float2(-mr[j], -mr[j]));
                  float2 e = make_float2(ex2(t.x), ex2(t.y));
                  float2 w = mul2(e, vf);
                  if constexpr (decltype(masked)::value) {
                    // a hidden key's codes and scales may hold anything
                    if (key0 + 32 * b + 8 * q >= lim[j]) e.x = w.x = 0.0f;
                    if (key0 + 32 * b + 8 * q + 1 >= lim[j]) e.y = w.y = 0.0f;
                  }
                  sum[j] = add2(sum[j], e);
                  pk[j >> 1][8 * b + 2 * q + (j & 1)] = pack_bf16(w);
                  pl[j >> 1][8 * b + 2 * q + (j & 1)] =
                      pack_rest(w, pk[j >> 1][8 * b + 2 * q + (j & 1)]);
                }
              }
            }
            bool fits = true;
#pragma unroll
            for (int j = 0; j < J; ++j) {
              sum[j].x += sum[j].y;
              fits = fits && sum[j].x < kSumMax;
            }
            if (!__all_sync(0xffffffffu, fits)) return false;
#pragma unroll
            for (int j = 0; j < J; ++j) l[j] += sum[j].x;
            put(pk, pl, all);
            return true;
          };
          const bool masked = k >= whole_tiles;
          bool fine = !rows;  // P of a warp without rows is whatever S was: no one reads its O
          if (rows && !(fresh && masked)) {
            if (fresh) {  // the first reference: the maximum of 16 keys
              uint32_t v[2][8];
              tmem_ld_16x256_x2(tu, v[0]);
              tmem_ld_16x256_x2(tu + kLow, v[1]);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int *s = reinterpret_cast<const int *>(v[j >> 1]) + 2 * (j & 1);
                float m = fmaxf(
                    fmaxf(static_cast<float>(s[0]) * ks[0].x, static_cast<float>(s[1]) * ks[0].y),
                    fmaxf(static_cast<float>(s[4]) * ks[4].x, static_cast<float>(s[5]) * ks[4].y));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                mr[j] = c[j] * fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
              }
            }
            const std::true_type yes{};
            const std::false_type no{};
            fine = narrow ? (masked ? pass(yes, no) : pass(no, no))
                          : (masked ? pass(yes, yes) : pass(no, yes));
            if (fresh && !fine)
#pragma unroll
              for (int j = 0; j < 4; ++j) mr[j] = -INFINITY;
          }
          if (!fine) {
            // Two passes, keys masked by row: the maximum first. The reference moves only where
            // the maximum passed it by 2^8, so that O is rarely rescaled.
            float mx[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) mx[j] = -INFINITY;
#pragma unroll 1
            for (int b = 0; b < 64; b += 16) {
              uint32_t v[2][8];
              tmem_ld_16x256_x2(tu + b, v[0]);
              tmem_ld_16x256_x2(tu + kLow + b, v[1]);
              tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float2 kf = ks[b / 2 + 4 * q];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int *s = reinterpret_cast<const int *>(v[j >> 1]) + 4 * q + 2 * (j & 1);
                  const float x0 = static_cast<float>(s[0]) * kf.x;
                  const float x1 = static_cast<float>(s[1]) * kf.y;
                  if (key0 + b + 8 * q < lim[j]) mx[j] = fmaxf(mx[j], x0);
                  if (key0 + b + 8 * q + 1 < lim[j]) mx[j] = fmaxf(mx[j], x1);
                }
              }
            }
            float al[4];
            bool moved = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
              mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
              const float tm = mx[j] == -INFINITY ? -INFINITY : c[j] * mx[j];
              const bool move = tm > -INFINITY && (mr[j] == -INFINITY || tm - mr[j] > 8.0f);
              al[j] = move && mr[j] != -INFINITY ? ex2(mr[j] - tm) : 1.0f;
              if (move) mr[j] = tm;
              l[j] *= al[j];
              moved = moved || move;
            }
            if (__any_sync(0xffffffffu, moved) && !fresh) {
              // the product before this half tile must be in O before O is rescaled
              if (!wait(&pvin[2 * hf + (h ^ 1)], h ? par : par ^ 1)) break;
              tc_fence_after();
#pragma unroll 1
              for (int q = 0; q < 16; ++q) {
                uint32_t v[8];
                tmem_ld_16x256_x1(to + 8 * q, v);
                tmem_ld_16x256_x1(to + kLow + 8 * q, v + 4);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  v[j] = __float_as_uint(__uint_as_float(v[j]) * al[j >> 1]);
                tmem_st_16x256_x1(to + 8 * q, v);
                tmem_st_16x256_x1(to + kLow + 8 * q, v + 4);
              }
            }
            uint32_t pk[2][16], pl[2][16];
#pragma unroll
            for (int b = 0; b < 64; b += 16) {
              uint32_t v[2][8];
              tmem_ld_16x256_x2(tu + b, v[0]);
              tmem_ld_16x256_x2(tu + kLow + b, v[1]);
              tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float2 kf = ks[b / 2 + 4 * q], vf = vs[b / 2 + 4 * q];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int *s = reinterpret_cast<const int *>(v[j >> 1]) + 4 * q + 2 * (j & 1);
                  const float nm = mr[j] == -INFINITY ? 0.0f : -mr[j];
                  const float x0 = static_cast<float>(s[0]) * kf.x;
                  const float x1 = static_cast<float>(s[1]) * kf.y;
                  const bool s0 = key0 + b + 8 * q < lim[j], s1 = key0 + b + 8 * q + 1 < lim[j];
                  const float e0 = s0 ? ex2(fmaf(x0, c[j], nm)) : 0.0f;
                  const float e1 = s1 ? ex2(fmaf(x1, c[j], nm)) : 0.0f;
                  l[j] += e0 + e1;
                  const float2 w = make_float2(s0 ? e0 * vf.x : 0.0f, s1 ? e1 * vf.y : 0.0f);
                  const int at = b / 4 + 2 * q + (j & 1);
                  pk[j >> 1][at] = pack_bf16(w);
                  pl[j >> 1][at] = pack_rest(w, pk[j >> 1][at]);
                }
              }
            }
            put(pk, pl, std::true_type{});
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&pfull[2 * hf + h]);
            if (h == 1) mbar_arrive_n(&empty[st], step);  // for the other group too where split
          }
          fresh = false;
        }
      }
      if (!ok) break;
      kt += k1 - k0;
      // ---- the piece's result ----
      const bool mine = !fresh;  // this group took some key tile
      if (mine) {
        if (!wait(&ofull[hf], np & 1)) break;
        ++np;
        tc_fence_after();
      }
      // from here on a lane has one row: its sum and reference come from the lanes 4 (r % 8)
      float lr = 0.0f, rm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float s = l[j];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s = __shfl_sync(0xffffffffu, s, 4 * (lane & 7));
        const float m = __shfl_sync(0xffffffffu, mr[j], 4 * (lane & 7));
        if (lane >> 3 == j) lr = s, rm = m;
      }
      const int row = 32 * (warp & 3) + lane;
      float wa = 1.0f, wb = 0.0f;  // weights of A's and B's O
      if (split && k1 > k0 + 1) {
        // both groups took key tiles of the same rows: A joins B's sums and reads B's O
        if (hf == 1) {
          bsum[2 * row] = rm;
          bsum[2 * row + 1] = lr;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bdone);
          if (!wait(btaken, nsp & 1)) break;
          tc_fence_after();
        } else {
          if (!wait(bdone, nsp & 1)) break;
          tc_fence_after();
          const float mb = bsum[2 * row], lb = bsum[2 * row + 1], m = fmaxf(rm, mb);
          if (m != -INFINITY) {
            wa = rm == m ? 1.0f : ex2(rm - m);
            wb = mb == m ? 1.0f : ex2(mb - m);
          }
          lr = (wa == 0.0f ? 0.0f : wa * lr) + (wb == 0.0f ? 0.0f : wb * lb);
          rm = m;
        }
        ++nsp;
      }
      if (split ? hf == 0 : pc->ntok > hf * a.TA) {
        const bool whole = pc->starts && pc->ends;
        int tok, head;
        const bool valid = place(a, pc->ntok, row, &tok, &head) && tok0 + tok < pc->ntok;
        const bool join = split && k1 > k0 + 1;
        const int slot = 2 * blockIdx.x + (pc->starts ? 1 : 0);
        const float inv = 1.0f / lr;  // not used where lr is 0
        T *orow = static_cast<T *>(a.out) + (valid ? q_row(tok, head) : 0) * kHd;
        float *prow = a.po + slot * slot_o + ((tok0 ? kRows : 0) + row) * kHd;
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          uint32_t v[32];
          if (mine) {
            tmem_ld32(to + 32 * b, v);
            tmem_wait_ld();
          }
          if (join) {
            uint32_t u[32];
            tmem_ld32(to + 128 + 32 * b, u);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float z = wa == 0.0f ? 0.0f : wa * __uint_as_float(v[j]);
              if (wb != 0.0f) z = fmaf(wb, __uint_as_float(u[j]), z);
              v[j] = __float_as_uint(z);
            }
          }
          if (!valid) continue;
          if (whole) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              T o[8];
#pragma unroll
              for (int u = 0; u < 8; ++u)  // a row that sees no key: zero
                o[u] = from_f32<T>(lr == 0.0f ? 0.0f : __uint_as_float(v[j + u]) * inv);
              uint4 raw;
              memcpy(&raw, o, 16);
              *reinterpret_cast<uint4 *>(orow + 32 * b + j) = raw;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<uint4 *>(prow + 32 * b + j) =
                  make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
        tc_fence_before();
        if (!whole && valid) {
          float *ml = a.ml + slot * slot_ml + ((tok0 ? kRows : 0) + row) * 2;
          ml[0] = rm;
          ml[1] = lr;
        }
        if (join) {
          __syncwarp();
          if (lane == 0) mbar_arrive(btaken);
        }
      }
      done();
    }
  } else if (warp < 12) {
    // --------------------------------------------------------------- V codes to bf16 ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(80));
    const int ct = threadIdx.x - 256;
    const int ch = ct & 7, key0 = ct >> 3;  // 16-byte chunk, first key; keys step by 16
    int kt = 0;
    bool ok = true;
    while (const Piece *pc = next()) {
      for (int k = pc->k0; k < pc->k1; ++k, ++kt) {
        const int st = kt % kStages, vb = kt & 1;
        ok = bar_wait(&vland[st], (kt / kStages) & 1, abort_flag, status) &&
             bar_wait(&vempty[vb], ((kt >> 1) & 1) ^ 1, abort_flag, status);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        const uint8_t *src = sm + st * kStage + kTile + key0 * kHd + ch * 16;
        uint8_t *dst = sm + kOffVs + vb * kV16 + (ch >> 2) * 16384 + key0 * 128;
        const int un = (ch & 3) * 2, sw = key0 & 7;  // keys step by 16: the swizzle stays
        // the chunks of panel 1 store their halves in the other order: banks stay apart
        const int f = ch >> 2;
        uint8_t *d0 = dst + ((un + f) ^ sw) * 16, *d1 = dst + ((un + 1 - f) ^ sw) * 16;
        const uint8_t *s0 = src + 8 * f, *s1 = src + 8 - 8 * f;
#pragma unroll 4
        for (int i = 0; i < 8; ++i) {
          const uint2 a0 = *reinterpret_cast<const uint2 *>(s0 + i * 16 * kHd);
          const uint2 a1 = *reinterpret_cast<const uint2 *>(s1 + i * 16 * kHd);
          const uint4 q = make_uint4(a0.x, a0.y, a1.x, a1.y);
          uint4 lo, hi;
          lo.x = codes_bf16(__byte_perm(q.x, 0, 0x4140));
          lo.y = codes_bf16(__byte_perm(q.x, 0, 0x4342));
          lo.z = codes_bf16(__byte_perm(q.y, 0, 0x4140));
          lo.w = codes_bf16(__byte_perm(q.y, 0, 0x4342));
          hi.x = codes_bf16(__byte_perm(q.z, 0, 0x4140));
          hi.y = codes_bf16(__byte_perm(q.z, 0, 0x4342));
          hi.z = codes_bf16(__byte_perm(q.w, 0, 0x4140));
          hi.w = codes_bf16(__byte_perm(q.w, 0, 0x4342));
          *reinterpret_cast<uint4 *>(d0 + i * 16 * 128) = lo;
          *reinterpret_cast<uint4 *>(d1 + i * 16 * 128) = hi;
        }
        fence_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&vfull[vb]);
          mbar_arrive(&empty[st]);
        }
      }
      if (!ok) break;
      done();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(80));
    if (warp < 14) {
      // ----------------------------------------------------------------- MMA issuers ----
      // All lanes walk the tiles, one elected lane issues: descriptors then stay in uniform
      // registers (in code under `lane == 0` every MMA paid for moving them there, 100 to 190
      // cycles an MMA against its 65). The group's S is two half tiles of 64 keys: while the softmax
      // is at one, the other's P V and the next tile's S in its place run here.
      constexpr uint32_t id_s = i8_idesc(128, 64);
      const int hf = warp - 12;
      const bool lead = elect_one();
      const uint64_t qd = sw128_desc(smem_u32(sm + kOffQ));
      const uint64_t kd0 = sw128_desc(smem_u32(sm)), vd0 = v16_desc(smem_u32(sm + kOffVs));
      const uint32_t tmem_s = tmem + 128 * hf, tmem_o = tmem + 256 + 128 * hf;
      int kt = 0, np = 0, nt = 0;  // tiles before the piece, pieces, this group's tiles
      bool ok = true;
      auto wait = [&](uint64_t *bar, int parity) {
        ok = __all_sync(0xffffffffu, bar_wait(bar, parity, abort_flag, status));
        tc_fence_after();
        return ok;
      };
      while (const Piece *pc = next()) {
        const int n = __shfl_sync(0xffffffffu, pc->k1 - pc->k0, 0);
        const bool split = __shfl_sync(0xffffffffu, pc->ntok, 0) <= a.TA;
        done();
        if (n <= 0) continue;
        if (!wait(qfull, np & 1)) break;
        ++np;
        // a split piece's tile has one reader, which answers for two
        const int step = split ? 2 : 1;
        const uint64_t q = qd + (split ? 0 : hf) * (kTile >> 4);
        auto scores = [&](int j, int h) {  // by the elected lane; K of tile j is there
          const uint64_t kd = kd0 + (j % kStages) * (kStage >> 4) + h * (kTile >> 5);
          const uint32_t d = tmem_s + 64 * h;
          mma_i8(d, q, kd, id_s, 0);
#pragma unroll
          for (int x = 1; x < kHd / 32; ++x) mma_i8(d, q + 2 * x, kd + 2 * x, id_s, 1);
          mma_commit(&sfull[2 * hf + h]);
          mbar_arrive(&sfull[2 * hf + h]);  // passes on what `full` showed: the scales are there
          if (h == 1) {
            mma_commit(&empty[j % kStages]);
            if (split) mma_commit(&empty[j % kStages]);
          }
        };
        auto keys_there = [&](int j) {
          const bool got = wait(&full[j % kFull], (j / kFull) & 1);
          if (!a.copies) fence_async();  // K was written by plain copies
          return got;
        };
        int i = split ? hf : 0;
        if (i < n) {
          if (!keys_there(kt + i)) break;
          if (lead) {
            scores(kt + i, 0);
            scores(kt + i, 1);
          }
          __syncwarp();
        }
        // After this group's last scores the next piece's queries may come (released after the
        // products, they held up V's pages too: 98 us, not 84, for 64 sequences of 4 draft rows
        // over 2K keys). The products begin when
        // both groups' of the piece before have ended: a group that had no tile there would
        // otherwise wait for a bf16 V buffer two fills ahead, and a parity tells only one.
        if (lead && i + step >= n) mma_commit(qempty);
        __syncwarp();
        if (np > 1 && !wait(pdone, np & 1)) break;
#pragma unroll 1
        for (uint32_t acc = 0; ok && i < n; i += step, ++nt) {
          const int j = kt + i, vb = j & 1;
          const bool more = i + step < n;
          if (!wait(&vfull[vb], (j >> 1) & 1)) break;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            if (h == 0 && more && !keys_there(j + step)) break;
            if (!wait(&pfull[2 * hf + h], nt & 1)) break;
            if (lead) {
              const uint64_t vd = vd0 + vb * (kV16 >> 4) + h * (4 * 2048 >> 4);
              const uint32_t pa = tmem_s + 64 * h;
              mma_bf16_ts(tmem_o, pa, vd, kIdescPv, acc);  // a piece's first overwrites O
#pragma unroll
              for (int x = 1; x < 4; ++x)
                mma_bf16_ts(tmem_o, pa + 8 * x, vd + x * (2048 >> 4), kIdescPv, 1);
#pragma unroll
              for (int x = 0; x < 4; ++x)  // the weights' second terms
                mma_bf16_ts(tmem_o, pa + 32 + 8 * x, vd + x * (2048 >> 4), kIdescPv, 1);
              mma_commit(&pvin[2 * hf + h]);
              if (more) scores(j + step, h);
              if (h == 1) {
                if (more && i + 2 * step >= n) mma_commit(qempty);
                mma_commit(&vempty[vb]);
                if (split) mma_commit(&vempty[vb]);
                if (!more) mma_commit(&ofull[hf]);
              }
            }
            __syncwarp();
            acc = 1;
          }
        }
        if (!ok) break;
        if (lead) mma_commit(pdone);
        __syncwarp();
        kt += n;
      }
      if (lead) {
        // nothing may read shared memory or write TMEM any more when they are given back
        mma_commit(&drained[hf]);
        mbar_drain(&drained[hf], 0);
      }
      __syncwarp();
    } else {
      // ------------------------------------ the walk, K pages and scales; Q and V pages ----
      const bool vwarp = warp == 15;
      const int bs = 1 << a.bs_log2;
      Walk w;
      w.s = first[0];
      w.g = first[1];
      w.t = first[2];
      w.off = first[3];
      w.left = static_cast<int>(run[1] - run[0]);
      int kt = 0, np = 0;
      bool ok = true;
      while (true) {
        const Piece *pc;
        if (vwarp) {
          pc = next();
          if (!pc) break;
        } else {
          ok = bar_wait(&aempty[na % kPieces], ((na / kPieces) & 1) ^ 1, abort_flag, status);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          Piece *p = &pieces[na % kPieces];
          if (lane == 0) {
            w.next(tab, a, p);
            if (p->valid && p->starts && !p->ends) {
              // the pieces of this item run up to the CTA that holds its last unit
              Meta &me = meta[blockIdx.x];
              me.t0 = p->t0;
              me.ntok = p->ntok;
              me.g = p->g;
              me.last = static_cast<int>(((run[1] + p->behind) * ctas - 1) / W);
              me.valid = 1;
            }
            mbar_arrive(&afull[na % kPieces]);
          }
          __syncwarp();
          ++na;
          if (!p->valid) break;
          pc = p;
        }
        const int32_t *bt = a.bt + static_cast<size_t>(pc->s) * a.max_blocks;
        const int keys = pc->keys, g = pc->g, k0 = pc->k0, k1 = pc->k1;
        if (vwarp) {
          const int t0 = pc->t0, ntok = pc->ntok, both = ntok > a.TA;
          done();
          if (k1 > k0) {
            // a tile's rows are TA tokens x G heads, which one box of the queries holds in order
            ok = bar_wait(qempty, (np & 1) ^ 1, abort_flag, status);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            if (ntok <= 4 * a.TN) {  // narrow: TN tokens at the first rows of each softmax warp
              if (lane == 0) {
                const int warps = (ntok + a.TN - 1) / a.TN;
                mbar_expect_tx(qfull, warps * a.TN * a.G * kHd);
                for (int i = 0; i < warps; ++i)
                  tma_load_3d(sm + kOffQ + i * 32 * kHd, &map_qn, 0, g * a.G, t0 + i * a.TN, qfull);
              }
            } else if (lane == 0) {
              mbar_expect_tx(qfull, (1 + both) * a.TA * a.G * kHd);
              tma_load_3d(sm + kOffQ, &map_q, 0, g * a.G, t0, qfull);
              if (both) tma_load_3d(sm + kOffQ + kTile, &map_q, 0, g * a.G, t0 + a.TA, qfull);
            }
            __syncwarp();
            ++np;
          }
        }
        // the page of position pos, as its first row in the pool; -1 behind the keys
        auto page_row = [&](int pos) -> long long {
          if (pos >= keys) return -1;
          int blk = __ldg(bt + (pos >> a.bs_log2));
          if (static_cast<uint32_t>(blk) >= static_cast<uint32_t>(a.num_blocks)) {
            *status = S8B_ERR_ARG;  // a page that does not exist: page 0 stands in
            blk = 0;
          }
          return (static_cast<long long>(blk) * a.Hkv + g) << a.bs_log2;
        };
        if (a.copies) {
          // A page's rows of one kv head are contiguous: lane i moves the tile's i-th page, K by a
          // tensor copy (the MMA wants it swizzled), V by a plain one. One lane's copies cost
          // the warp some 80 cycles each, so the 32 chunks of 16 bytes of each scale array go by
          // one cp.async per lane.
          const int rows = min(bs, kKeys), pages = kKeys / rows;
          long long row = lane < pages ? page_row(k0 * kKeys + lane * rows) : -1;
#pragma unroll 1
          for (int k = k0; k < k1; ++k, ++kt) {
            const int st = kt % kStages, pos = k * kKeys + lane * rows;
            const long long at = row < 0 ? -1 : row + (pos & (bs - 1));
            // the next tile's page ids are on their way while this tile waits for its stage
            row = k + 1 < k1 && lane < pages ? page_row(pos + kKeys) : -1;
            ok = bar_wait(&empty[st], ((kt / kStages) & 1) ^ 1, abort_flag, status);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            uint8_t *base = sm + st * kStage;
            uint64_t *bar = vwarp ? &vland[st] : &full[kt % kFull];
            const int n = __popc(__ballot_sync(0xffffffffu, at >= 0));
            if (lane == 0) mbar_expect_tx(bar, n * rows * kHd);
            __syncwarp();
            if (vwarp) {
              if (at >= 0)
                bulk_load(base + kTile + lane * rows * kHd, a.vc + at * kHd, rows * kHd, bar);
            } else {
              if (at >= 0) tma_load_2d(base + lane * rows * kHd, &map_k, 0, static_cast<int>(at), bar);
              __syncwarp();
              const long long pg = __shfl_sync(0xffffffffu, at, 4 * lane / rows);
              if (pg >= 0) {
                const uint32_t sc = smem_u32(base + 2 * kTile) + 16 * lane;
                const long long s4 = pg + (4 * lane & (rows - 1));
                cp16(sc, a.ks + s4);
                cp16(sc + kKeys * 4, a.vs + s4);
              }
              cp_arrive(bar);
            }
          }
        } else {
          // Pages of 1, 2 or 4 keys (less than a swizzle atom), or scales off a 16-byte boundary:
          // 16-byte copies per row.
#pragma unroll 1
          for (int k = k0; k < k1; ++k, ++kt) {
            const int st = kt % kStages;
            ok = bar_wait(&empty[st], ((kt / kStages) & 1) ^ 1, abort_flag, status);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            const uint32_t base = smem_u32(sm + st * kStage);
            const int ch = lane & 7;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {  // rows 32 q + lane
              const int pos = k * kKeys + 32 * q + lane;
              long long at = page_row(pos);
              if (at >= 0) at += pos & (bs - 1);
              if (at >= 0 && !vwarp) {
                cp4(base + 2 * kTile + (32 * q + lane) * 4, a.ks + at);
                cp4(base + 2 * kTile + kKeys * 4 + (32 * q + lane) * 4, a.vs + at);
              }
#pragma unroll 2
              for (int j = 0; j < 8; ++j) {
                const int r = 32 * q + (lane >> 3) + 4 * j;
                const long long src = __shfl_sync(0xffffffffu, at, r & 31);
                const uint32_t dst = base + (vwarp ? kTile + r * kHd + ch * 16
                                                   : r * kHd + ((ch ^ (r & 7)) * 16));
                if (src >= 0) cp16(dst, (vwarp ? a.vc : a.kc) + src * kHd + ch * 16);
              }
            }
            cp_arrive(vwarp ? &vland[st] : &full[kt % kFull]);  // the MMA's warps fence for their proxy
          }
        }
        if (!ok) break;
      }
      // nothing may still be on its way when the shared memory goes
      if (a.copies)
        for (int i = max(0, kt - kStages); i < kt; ++i)
          if (vwarp) mbar_drain(&vland[i % kStages], (i / kStages) & 1);
          else mbar_drain(&full[i % kFull], (i / kFull) & 1);
      if (vwarp && np > 0) mbar_drain(qfull, (np - 1) & 1);
      cp_wait_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
}

// -------------------------------------------------------------------------------- merge ----
// Joins the pieces of an item that CTA boundaries split, in key order: grid (CTAs, row groups),
// one warp per row at a time; lanes are pieces while the weights are found (a pass over 32
// pieces at a time), then four output values each.
constexpr int kMergeWarps = 8, kMergeGroups = 16;
template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32) chunk_merge_kernel(const ChunkArgs a) {
  using namespace ca;
  griddep_launch();
  griddep_wait();
  const Meta me = reinterpret_cast<const Meta *>(a.ws + kOffMeta)[blockIdx.x];
  if (!me.valid) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x, n = me.last - c0 + 1;
  auto slot = [&](int i) { return static_cast<size_t>(2 * (c0 + i) + (i == 0)); };
  for (int r = blockIdx.y * kMergeWarps + warp; r < kItemRows; r += gridDim.y * kMergeWarps) {
    int tok, head;
    const bool is = place(a, me.ntok, r & 127, &tok, &head);
    const int i = (r >> 7) * a.TA + tok;
    if (!is || i >= me.ntok) continue;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = 0; b < n; b += 32) {
      float mi = -INFINITY, li = 0.0f;
      if (b + lane < n) {
        const float2 v = *reinterpret_cast<const float2 *>(a.ml + slot(b + lane) * slot_ml + r * 2);
        mi = v.x, li = v.y;
      }
      const float mb = fmaxf(m, warp_max(mi));
      // a piece of which the row sees no key has no weight, and nothing of it is read
      const float w = mi == -INFINITY ? 0.0f : mi == mb ? 1.0f : ex2(mi - mb);
      const float old = m == -INFINITY ? 0.0f : m == mb ? 1.0f : ex2(m - mb);
      m = mb;
      float s = w == 0.0f ? 0.0f : w * li;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      l = old * l + s;
#pragma unroll
      for (int x = 0; x < 4; ++x) o[x] *= old;
      const int nb = min(32, n - b);
#pragma unroll 4
      for (int x = 0; x < nb; ++x) {
        const float wx = __shfl_sync(0xffffffffu, w, x);
        if (wx == 0.0f) continue;
        const float4 v = *reinterpret_cast<const float4 *>(a.po + slot(b + x) * slot_o + r * kHd +
                                                            4 * lane);
        o[0] += wx * v.x;
        o[1] += wx * v.y;
        o[2] += wx * v.z;
        o[3] += wx * v.w;
      }
    }
    const float inv = 1.0f / l;  // not used where l is 0
    T t[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) t[x] = from_f32<T>(l == 0.0f ? 0.0f : o[x] * inv);
    uint2 raw;
    memcpy(&raw, t, 8);
    const size_t qrow = static_cast<size_t>(me.t0 + i) * a.Hq + me.g * a.G + head;
    *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + qrow * kHd + 4 * lane) = raw;
  }
}

// 3-D map over the queries [T][Hq][128 B], box {128, G, TA}: a tile's rows in order.
int make_map_q(CUtensorMap *map, const int8_t *q, int T, int Hq, int G, int TA) {
  auto fn = encode_fn();
  if (!fn) return S8B_ERR_CUDA;
  const cuuint64_t dims[3] = {ca::kHd, static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {ca::kHd, static_cast<cuuint64_t>(Hq) * ca::kHd};
  const cuuint32_t box[3] = {ca::kHd, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(TA)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t *>(q), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? S8B_OK : S8B_ERR_ALIGN;
}

template <typename T>
cudaError_t launch_attn(int ctas, cudaStream_t st, const CUtensorMap &map_k,
                        const CUtensorMap &map_q, const CUtensorMap &map_qn,
                        const ChunkArgs &a) {
  ensure_smem(reinterpret_cast<const void *>(chunk_attn_kernel<T>), ca::kSmem);
  return launch_pdl(chunk_attn_kernel<T>, dim3(ctas), dim3(ca::kThreads), ca::kSmem, st,
                    map_k, map_q, map_qn, a);
}

int chunk_ctas() { return min(sm_count(), ca::kMaxCtas); }

}  // namespace
}  // namespace s8b

using namespace s8b;

extern "C" size_t s8b_paged_chunk_workspace_size(void) {
  using namespace ca;
  return kOffMl + static_cast<size_t>(2 * chunk_ctas()) * (slot_ml + slot_o) * sizeof(float);
}

extern "C" int s8b_paged_chunk_q8(const int8_t *q_i8, const float *q_s, const int8_t *kc,
                                  const float *ks, const int8_t *vc, const float *vs,
                                  const int32_t *block_table, const int32_t *context_lens,
                                  const int32_t *cu_q, void *out, int T_, int S, int Hq, int Hkv,
                                  int D, int block_size, int max_blocks, int num_blocks,
                                  float scale, void *workspace, size_t workspace_bytes, int dtype,
                                  void *stream) {
  using namespace ca;
  if (!q_i8 || !q_s || !kc || !ks || !vc || !vs || !block_table || !context_lens || !cu_q || !out)
    return S8B_ERR_ARG;
  if (!(scale > 0.0f) || scale > 1e30f) return S8B_ERR_ARG;
  if (dtype != S8B_BF16 && dtype != S8B_FP16) return S8B_ERR_DTYPE;
  if (T_ < 0 || S < 0 || S > kMaxSeqs || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq / Hkv > kRows ||
      D != kHd || max_blocks <= 0 || num_blocks <= 0)
    return S8B_ERR_SHAPE;
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size && bs_log2 < 8) ++bs_log2;
  if (block_size != (1 << bs_log2)) return S8B_ERR_SHAPE;
  // rows of the pool and rows x heads of the queries are counted in 32 bits
  if (static_cast<unsigned long long>(num_blocks) * Hkv * block_size >= 0xffffffffull ||
      static_cast<long long>(T_) * Hq > 0x7fffffffll)
    return S8B_ERR_SHAPE;
  if (!aligned(q_i8, 16) || !aligned(kc, 16) || !aligned(vc, 16) || !aligned(out, 16) ||
      !aligned(ks, 4) || !aligned(vs, 4) || !aligned(q_s, 4) || !aligned(block_table, 4) ||
      !aligned(context_lens, 4) || !aligned(cu_q, 4))
    return S8B_ERR_ALIGN;
  if (T_ == 0 || S == 0) return S8B_OK;
  if (!workspace || workspace_bytes < s8b_paged_chunk_workspace_size()) return S8B_ERR_WORKSPACE;
  if (!aligned(workspace, 256)) return S8B_ERR_ALIGN;
  ChunkArgs a = {};
  a.q = q_i8;
  a.qs = q_s;
  a.kc = kc;
  a.vc = vc;
  a.ks = ks;
  a.vs = vs;
  a.bt = block_table;
  a.ctx = context_lens;
  a.cu = cu_q;
  a.out = out;
  a.ws = static_cast<uint8_t *>(workspace);
  const int ctas = chunk_ctas();
  a.ml = reinterpret_cast<float *>(a.ws + kOffMl);
  a.po = a.ml + static_cast<size_t>(2 * ctas) * slot_ml;
  a.T = T_;
  a.S = S;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.TA = kRows / a.G;
  a.TN = a.G <= 8 ? 8 / a.G : 0;
  a.bs_log2 = bs_log2;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  const long long reach = static_cast<long long>(max_blocks) << bs_log2;
  a.cap = static_cast<int>(reach < 0x7fffff00ll ? reach : 0x7fffff00ll);
  a.c = scale * 1.4426950408889634f;
  const cudaStream_t st = (cudaStream_t)stream;
  // bulk copies want 16-byte boundaries, the tensor copy whole 8-row swizzle atoms and row
  // numbers below 2^31
  const unsigned long long rows = static_cast<unsigned long long>(num_blocks) * Hkv * block_size;
  CUtensorMap map_k, map_q, map_qn;
  memset(&map_k, 0, sizeof(map_k));
  if (const int rc = make_map_q(&map_q, q_i8, T_, Hq, a.G, a.TA)) return rc;
  map_qn = map_q;
  if (a.TN > 0)
    if (const int rc = make_map_q(&map_qn, q_i8, T_, Hq, a.G, a.TN)) return rc;
  a.copies = block_size >= 8 && aligned(ks, 16) && aligned(vs, 16) && rows < (1ull << 31);
  if (a.copies) {
    const int rc =
        make_map_2d(&map_k, kc, kHd, rows, kHd, kHd, block_size < kKeys ? block_size : kKeys);
    if (rc) return rc;
  }
  S8B_DISPATCH_DTYPE(dtype, T, {
    cudaError_t e = launch_attn<T>(ctas, st, map_k, map_q, map_qn, a);
    if (e == cudaSuccess)
      e = launch_pdl(chunk_merge_kernel<T>, dim3(ctas, kMergeGroups), dim3(kMergeWarps * 32), 0,
                     st, a);
    if (e != cudaSuccess) {
      record_cuda_error(e);
      return S8B_ERR_CUDA;
    }
  });
  return check_launch(2);
}
