// Attention over the paged 8-bit KV cache on sm_100a: the form for many query rows (prompts, chunks,
// wide groups of heads). The formula and the masks are paged_attn.cu's.
//
// k_paged_tile: an item is 256 rows of one (sequence, KV head) -- its tokens times the query heads of the
// group, token-major, so every head of the group uses a key tile once -- as two 128-row tiles. The bound is
// the tensor core (S = Q K^T and O = P V, tcgen05 kind::f16) against the exponentials (one each score).
// Roles of a CTA (one per SM, 16 warps; registers go from the others to the softmax: with 144 and 112 the third
// case below takes 221 us, with 152 and 96 or 112 225, with 128 for all, and spills, 224):
//   warps 0-3, 4-7   the softmax of the first and second 128 rows, a row a thread, 64 keys a step: scores from
//                    TMEM, the running maximum and sum in float32 registers, weights back to TMEM as fp16 over
//                    the scores that they came from. They also fetch the queries and write the output.
//   warps 8-11       pages to operands: 128 keys of int8 from HBM through registers (a tile ahead) to 16 bits
//                    in shared memory (exact: keys in the queries' type, values in fp16), two stages of each.
//                    No scale is multiplied in: the key scale multiplies the score, the value scale the weight.
//   warps 12, 15     one thread each issues the products of a row tile: a step's P V, then the scores that the
//                    same 64 columns of TMEM hold next, while the softmax works on the other 64. (One warp for
//                    both row tiles waited for one while the other's weights were ready: 8 prompts of 2048, 16
//                    heads on 8, took 257 us instead of 236.)
//   warp 13          walks the line (below) and hands the pieces to the others.
//   warp 14          looks the tiles' pages and their scales up, up to four tiles ahead.
// O stays in TMEM, in units of the row's own largest contribution: with m the running maximum of its scores (log2)
// and v that of score + log2 s_v, over the keys that the row itself sees, a key's weight is 2^(score - m) s_v
// 2^(m - v + 10). O is rescaled only when m or v grew by more than 4, which is rare after an item's first tile; so
// weights stay below 2^14 in fp16 and keep 11 bits down to 2^-24 of the largest contribution, whatever lies in pages
// that the mask hides from the row and however far apart the pages' scales are. (With one reference a tile, its largest
// value scale, rows lost bits to later pages, and values below 4e-34 became NaN.)
// Items lie on one line, cut into equal parts, one per SM, as in the few-row form; an item in several parts is
// joined by the last of them in key order. An item is as long as its key tiles and kItemCost = 2 more, for its
// queries, its output and its masked tiles: equal numbers of tiles left the SMs with many short items
// longest (with 0, 1, 2 and 3 more: 8 prompts of 2048, 16 heads on 8, 204, 196, 195 and 199 us; 8192 tokens with a
// window of 2048, 32 heads on 8, 361, 332, 313 and 315).
//
// Measured on B200 (a graph of calls): 8 prompts of 2048, 16 heads on 8, bf16: 195 us, 0.71 PFLOP/s of visible
// products; 8192 with a window of 2048, 32 heads on 8: 312 us, 0.77; 4 chunks of 512 at the end of up to 12289,
// 32 heads on 8, fp16: 221 us, 0.89. No unit is full: in a steady tile of 4,800 cycles the tensor pipe runs
// 2,700 (64 keys a product read Q from shared memory twice as often as 128 do: 54 cycles instead of 32 for 64),
// the exponentials' pipe 2,000, the shared-memory pipe 3,800 and each scheduler issues 2,400 instructions.
// Scores of 128 keys a product read less but leave one score buffer a row tile, so that the softmax waits for
// them: 229, 409 and 254 us.
#include <algorithm>
#include <cfloat>

#include "det_math.cuh"
#include "paged.cuh"
#include "uwc_host.h"

namespace {

using namespace paged;

constexpr int kRows = 128;                   // rows of a softmax warpgroup
constexpr int kTile = 128;                   // keys per tile
constexpr int kGroups = kTile / 16;          // 16-key groups, each inside one page
constexpr int kThreads = 16 * 32;
constexpr int kHalf = kTile * 128;           // bytes of 128 rows x 64 dims of fp16 (one swizzled block)
constexpr int kOperand = 2 * kHalf;          // a 128 x 128 fp16 operand
constexpr int kAhead = 4;                    // tiles whose pages are looked up ahead of their loads
constexpr int kPageRing = 8;                 // slots: those, and up to four that the softmax still reads scales of
constexpr int kSeqs = 1024;                  // sequences whose span and tiles are kept in shared memory
constexpr int kSmem = 1024 + 6 * kOperand + kSeqs * 24;   // two query tiles, two stages of keys, two of values
constexpr int kMinTiles = 4;                 // a CTA's least share of the line
constexpr int kItemCost = 2;                 // what an item costs beside its tiles, in tiles
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
// 128 dims; values are stored key by key: B is MN-major
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((uint32_t)(kHd >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
constexpr float kNoScore = 1.4e-45f;         // the factor of scores in pages of (almost) zero keys: not 0, so that -inf stays
                                             // -inf, and the smallest there is, since a bf16 query may reach 1e38
constexpr float kRaise = 4.f;                // log2 by which a score may pass the running maximum
constexpr float kUnit = 10.f;                // log2 of the largest contribution's fp16 weight when v was set
constexpr float kLow = 116.f;                // v is no lower than m by more: 2^(m - v + kUnit) is finite, 2^(v - m - kUnit) not 0

struct TileArgs {
  AttnArgs a;
  float* part_o;           // (2 grid, 2, 32, 128, 4): a CTA's two partial items by row tile, four columns, row; unnormalized
  float2* part_ml;         // (2 grid, 256): running maximum (log2), sum
  uint32_t* counters;      // (grid, 2): finished parts of the item that starts in this CTA; the last brings it back to zero
  int withhold;            // 1: every other CTA looks no pages up (a test's hook), so that its waits run out
};

// 256 rows of one (sequence, KV head): tokens t0 .. t1 have rows in it.
struct Item : Keys<kTile> {
  __device__ __forceinline__ Item(const AttnArgs& a, const Span& sp, int G, int blk)
      : Keys<kTile>(a, sp, 2 * kRows * blk / G, min(sp.n - 1, (2 * kRows * blk + 2 * kRows - 1) / G)) {}
};

// The batch as a CTA's roles see it: spans and tiles (of one KV head) of the first kSeqs sequences in
// shared memory, of any further ones from global memory.
struct Batch {
  const AttnArgs& a;
  int G;
  int4* span_;             // row0, n, start, idle
  long long* tiles_;
  __device__ __forceinline__ Span span(int s) const {
    if (s >= kSeqs) return span_of(a.b, a.c.ps, s);
    const int4 x = span_[s];
    return Span{x.x, x.y, x.z, x.w != 0, false};
  }
  __device__ __forceinline__ int blocks(const Span& z) const { return (int)(((long long)z.n * G + 2 * kRows - 1) / (2 * kRows)); }
  // all lanes of a warp together
  __device__ __forceinline__ long long count(const Span& z) const {
    const int nb = blocks(z);
    long long t = 0;
#pragma unroll 1
    for (int b = threadIdx.x & 31; b < nb; b += 32) t += kItemCost + Item(a, z, G, b).total;
    return warp_sumll(t);
  }
  __device__ __forceinline__ long long tiles(int s) const { return s < kSeqs ? tiles_[s] : count(span(s)); }
  __device__ __forceinline__ void load() {
    const int n = min(a.b.seqs, kSeqs);
#pragma unroll 1
    for (int s = threadIdx.x; s < n; s += kThreads) {
      const Span z = span_of(a.b, a.c.ps, s);
      if (z.bad && blockIdx.x == 0) set_status(a.status, UWC_DEV_RANGE);
      span_[s] = make_int4(z.row0, z.n, z.start, z.idle);
    }
    if (blockIdx.x == 0)
#pragma unroll 1
      for (int s = kSeqs + threadIdx.x; s < a.b.seqs; s += kThreads)
        if (span_of(a.b, a.c.ps, s).bad) set_status(a.status, UWC_DEV_RANGE);
    __syncthreads();
#pragma unroll 1
    for (int s = threadIdx.x / 32; s < n; s += kThreads / 32) {
      const long long t = count(span(s));
      if ((threadIdx.x & 31) == 0) tiles_[s] = t;
    }
  }
};

// A CTA's part of the line: `left` units from unit u0 of block blk of KV head h of sequence s on. An item's units
// are kItemCost for itself and one a key tile.
struct Start {
  int s, h, blk, u0;
  int left, per;
};
// One warp, all lanes together.
__device__ __forceinline__ Start find_start(const Batch& q) {
  const int lane = threadIdx.x & 31, S = q.a.b.seqs, kept = min(S, kSeqs), Hkv = q.a.c.Hkv;
  long long sum = 0;
#pragma unroll 1
  for (int i = lane; i < kept; i += 32) sum += q.tiles_[i];
  sum = warp_sumll(sum);
#pragma unroll 1
  for (int i = kept; i < S; i++) sum += q.tiles(i);
  sum *= Hkv;
  Start p = {};
  // no less than an even share (a division of 64 bits is long code): grid * per >= sum
  p.per = max(kMinTiles, (int)((float)sum / (float)gridDim.x * 1.000001f) + 1);
  long long rest = (long long)p.per * blockIdx.x;
  p.left = (int)max(0ll, min((long long)p.per, sum - rest));
  if (p.left == 0) return p;
#pragma unroll 1
  for (; p.s < S; p.s++) {
    const long long one = q.tiles(p.s);
    if (rest < one * Hkv) {
      const Span sp = q.span(p.s);
      const int blks = q.blocks(sp);
#pragma unroll 1
      for (; rest >= one; p.h++) rest -= one;
#pragma unroll 1
      for (int b0 = 0; b0 < blks; b0 += 32) {
        const int t = b0 + lane < blks ? kItemCost + Item(q.a, sp, q.G, b0 + lane).total : 0;
        int inc = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > rest);
        if (hit) {
          const int l = __ffs(hit) - 1;
          p.blk = b0 + l;
          p.u0 = (int)(rest - __shfl_sync(0xffffffffu, inc - t, l));
          return p;
        }
        rest -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    rest -= one * Hkv;
  }
  p.left = 0;
  return p;
}

// One piece of it, inside one item, as the roles read it from shared memory.
struct Piece {
  int rows;                // rows of the item (0 ends the CTA's work), the first kRows of them warpgroup 0's
  int row0, first;         // the sequence's first row of the row tensors, the item's first row of the sequence
  int seq, head, start;    // start: -1 where the slot is idle
  int t0, t1, whole;       // tiles; whether they are the whole item
  int b0, b1;              // the CTAs that have parts of it
  int lo, hi, sink_end, tA, tB0;
  __device__ __forceinline__ int key(int i) const { return (i < tA ? i : tB0 + (i - tA)) * kTile; }
  __device__ __forceinline__ bool seen(int j, int n) const { return j < sink_end || (j < hi && j + n > lo); }
};
constexpr int kPieces = 4;   // pieces known ahead

// ---- tcgen05
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr) {
  // MN-major operand, 128-byte swizzle: 64 dims a 128-byte row, 8-key atoms 1024 bytes apart (SBO), the
  // next 64 dims one block on (LBO)
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(kHalf >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Two of four int8 values in the queries' type, exactly. bf16 has 8 significant bits, so the byte goes in
// parts: 0x4300 | its low seven bits is 128 + they, and 0x4300 | its top bit is 128, or 256 for a negative one.
__device__ __forceinline__ uint32_t i8_pair(uint32_t x, uint32_t sel, __half) { return i8_half2(x ^ 0x80808080u, sel); }
__device__ __forceinline__ uint32_t i8_pair(uint32_t x, uint32_t sel, __nv_bfloat16) {
  const uint32_t lo = __byte_perm(x & 0x7f7f7f7fu, 0x43434343u, sel), top = __byte_perm(x & 0x80808080u, 0x43434343u, sel);
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&top));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
struct IsBf16 { static constexpr uint32_t value = 0; };
template <>
struct IsBf16<__nv_bfloat16> { static constexpr uint32_t value = 1; };

// The n lowest bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int n) {
  uint32_t r;
  asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(r) : "r"(max(n, 0)));
  return r;
}

struct Bars {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], o_done[2][2], wg[2], piece_full[kPieces], piece_empty[kPieces], page_full[kAhead], page_empty[kAhead], fin;
};

// Pairs of float32 (one instruction for two), and the larger of three.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lo_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  return max3(__uint_as_float(a), __uint_as_float(b), __uint_as_float(c));
}
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) { return max3(a, __uint_as_float(b), __uint_as_float(c)); }

// Ends the role when a wait ran out; the other roles' waits then run out too.
#define TILE_WAIT(bar, parity) \
  if (!warp_wait(&(bar), (parity))) goto timeout

// A role's next piece, and its place in the ring given back.
#define TILE_PIECE(n)                                                                        \
  TILE_WAIT(bar.piece_full[(n) % kPieces], ((n) / kPieces) & 1);                             \
  const Piece& k = s_piece[(n) % kPieces];                                                   \
  if (k.rows == 0) break
#define TILE_PIECE_DONE(n)                                                                   \
  __syncwarp();                                                                              \
  if (lane == 0) mbar_arrive(&bar.piece_empty[(n) % kPieces])

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) k_paged_tile(const TileArgs ta) {
  const AttnArgs& a = ta.a;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bar;
  __shared__ Piece s_piece[kPieces];
  __shared__ __align__(16) float2 s_scale[kPageRing][kGroups];   // factor of scores (log2), value scale
  __shared__ __align__(16) float s_log[kPageRing][kGroups];      // log2 of the value scale
  __shared__ int s_unseen[kPageRing];              // 16-key groups that nobody sees
  __shared__ int s_row[kPageRing][kGroups];        // first cache row of the group's keys (-1: none; -2: no more tiles)
  __shared__ Start s_start;
  __shared__ uint32_t s_tmem;
  __shared__ int s_last[2];
  __shared__ int3 s_part[2];                       // the CTA's parts of items that others share: rows, b0, b1; [1]: starts here
  __shared__ int s_counted[2][2], s_gave_up;       // those that are counted, by row tile; whether a wait ran out
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smQ = smem_u32(sm), smK = smQ + 2 * kOperand, smV = smK + 2 * kOperand;
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&bar.q_full[i], 4);
      mbar_init(&bar.k_full[i], 4);
      mbar_init(&bar.k_empty[i], 2);
      mbar_init(&bar.v_full[i], 4);
      mbar_init(&bar.v_empty[i], 2);
      mbar_init(&bar.s_full[i][0], 2);
      mbar_init(&bar.s_full[i][1], 2);
      mbar_init(&bar.p_full[i][0], 4);
      mbar_init(&bar.p_full[i][1], 4);
      mbar_init(&bar.o_done[i][0], 1);
      mbar_init(&bar.o_done[i][1], 1);
      mbar_init(&bar.wg[i], 4);
    }
    mbar_init(&bar.fin, 2);
    s_counted[0][0] = s_counted[0][1] = s_counted[1][0] = s_counted[1][1] = s_gave_up = s_part[0].x = s_part[1].x = 0;
    for (int i = 0; i < kPieces; i++) {
      mbar_init(&bar.piece_full[i], 1);
      mbar_init(&bar.piece_empty[i], 11);
    }
    for (int i = 0; i < kAhead; i++) {
      mbar_init(&bar.page_full[i], 1);
      mbar_init(&bar.page_empty[i], 4);
    }
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  Batch batch{a, a.H / a.c.Hkv, reinterpret_cast<int4*>(sm + 6 * kOperand),
              reinterpret_cast<long long*>(sm + 6 * kOperand + kSeqs * 16)};
  batch.load();
  __syncthreads();
  if (warp == 0) {
    const Start p = find_start(batch);
    if (lane == 0) s_start = p;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int Hkv = a.c.Hkv, ps = a.c.ps, G = a.H / Hkv;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // ------------------------------------------------------------------ softmax, a row a thread
    const int w = warp >> 2, r = tid & (kRows - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128, tO = tmem + lanes + 256 + w * 128;
    const float inv_g = 1.0f / (float)G;
    uint32_t it = 0, all = 0, wgp = 0;             // this warpgroup's tiles, every tile, its barrier's phases
    // Row x of an item is token (x + rem) / G past the item's first one: a division of small numbers, exact in
    // float32 while they are below 2^20.
    auto token_of = [&](int x) { return (int)(((float)x + 0.5f) * inv_g); };
    const int dt = 2 / G, dh = 2 - dt * G;         // two rows on: tokens and heads of the group
    const long long by = dt * a.q_tok + dh * a.q_head, carry = a.q_tok - G * a.q_head;
    // Sends a piece's query rows on their way to this warp's part of the operand, two rows a step.
    auto fetch_q = [&](const Piece& k) {
      const int rows = min(kRows, k.rows - kRows * w);
      if (rows <= 0) return;
      const int r0 = 32 * (warp & 3) + (lane >> 4), tok = token_of(k.first - k.first / G * G + kRows * w + r0), c = lane & 15;
      int head = k.first - k.first / G * G + kRows * w + r0 - tok * G;
      const T* q = reinterpret_cast<const T*>(a.q) + (long long)(k.row0 + k.first / G + tok) * a.q_tok + (long long)(k.head * G + head) * a.q_head + 8 * c;
      const uint32_t at = smQ + w * kOperand + (c >> 3) * kHalf + r0 * 128;
#pragma unroll 4
      for (int x = 0; x < 32; x += 2) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + x * 128 + (((c & 7) ^ ((r0 + x) & 7)) << 4)),
                     "l"(r0 + x < rows ? q : reinterpret_cast<const T*>(a.q)), "r"(r0 + x < rows ? 16 : 0)
                     : "memory");
        q += by;
        head += dh;
        if (head >= G) {
          head -= G;
          q += carry;
        }
      }
    };
    TILE_WAIT(bar.piece_full[0], 0);
    fetch_q(s_piece[0]);
#pragma unroll 1
    for (uint32_t n = 0;; n++) {
      TILE_PIECE(n);
      const int rows = min(kRows, k.rows - kRows * w);
      if (rows <= 0) {                             // only w = 1: the second tile of a short item
        all += k.t1 - k.t0;
        TILE_WAIT(bar.piece_full[(n + 1) % kPieces], ((n + 1) / kPieces) & 1);
        fetch_q(s_piece[(n + 1) % kPieces]);
        TILE_PIECE_DONE(n);
        continue;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async_smem();
      warp_arrive(&bar.q_full[w]);
      const int tok0 = k.first / G, rem0 = k.first - tok0 * G;
      const int my_tok = token_of(kRows * w + r + rem0), my_head = kRows * w + r + rem0 - my_tok * G;
      const bool live = r < rows;
      const int pos = live && k.start >= 0 ? k.start + tok0 + my_tok : -1;
      // positions of this warpgroup's first and last row bound where its masks are needed
      const int pa = k.start < 0 ? -1 : k.start + tok0 + token_of(kRows * w + rem0);
      const int pb = k.start < 0 ? -1 : k.start + tok0 + token_of(kRows * w + rows - 1 + rem0);
      float m = kNoMax, v = kNoMax, l = 0.f, unit = 0.f;   // unit: 2^(m - v + kUnit)
      // 64 keys a step; the next step's scores are being computed meanwhile, in the other half of this row
      // tile's score columns
#pragma unroll 1
      for (int u = 2 * k.t0; u < 2 * k.t1; u++, it++) {
        const int h = u & 1, j0 = k.key(u >> 1) + 64 * h;
        const uint32_t tH = tS + 64 * h, slot = all % kPageRing;
        all += h;
        TILE_WAIT(bar.s_full[w][h], (it >> 1) & 1);
        tc_fence_after();
        uint32_t s0[32], s1[32];
        tmem_ld_32x32b_x32(tH, s0);
        float kf[4], vf[4];                        // the pages' factors for scores (log2) and values
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          const uint4 x = lds128(smem_u32(&s_scale[slot][4 * h + g]));
          kf[g] = __uint_as_float(x.x);
          vf[g] = __uint_as_float(x.y);
          kf[g + 1] = __uint_as_float(x.z);
          vf[g + 1] = __uint_as_float(x.w);
        }
        const uint4 lv = lds128(smem_u32(&s_log[slot][4 * h]));
        const int unseen = s_unseen[slot] >> (4 * h) & 15;
        // whether some key is hidden from some row: past its position, out of its window, without a page
        const bool hidden = j0 + 63 > pa || (a.window >= 0 && !(j0 > pb - a.window || j0 + 64 <= a.sinks)) || unseen;
        if (hidden) {
          if (j0 > pb || (a.window >= 0 && j0 + 63 <= pa - a.window && j0 >= a.sinks)) {
            // keys that none of these rows sees (the other row tile's): weights of zero. With a window of
            // 2048 that is one step in twenty: 338 us instead of 358 (8192 tokens, 32 heads on 8).
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; x++) s0[x] = 0;
            tmem_st_32x32b_x32(tH, s0);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&bar.p_full[w][h]);
            continue;
          }
          // only keys at an edge: their hidden scores become -inf where they are, in a rolled loop (every
          // instruction of the code around it is fetched for every step)
#pragma unroll 1
          for (int c = 0; c < 2; c++) {
            tmem_ld_32x32b_x32(tH + 32 * c, s0);
            tmem_wait_ld();
            const int last = pos - j0 - 32 * c, from = a.window < 0 ? -kTile : last - a.window, sink = a.sinks - j0 - 32 * c;
            const uint32_t pages = (unseen >> (2 * c) & 1 ? 0 : 0xffffu) | (unseen >> (2 * c + 1) & 1 ? 0 : 0xffff0000u);
            const uint32_t seen = low_bits(last + 1) & (~low_bits(from + 1) | low_bits(sink)) & pages;
#pragma unroll
            for (int x = 0; x < 32; x++) s0[x] = seen >> x & 1 ? s0[x] : 0xff800000u;
            tmem_st_32x32b_x32(tH + 32 * c, s0);
          }
          tmem_wait_st();
          tmem_ld_32x32b_x32(tH, s0);
        }
        float mx = kNoMax, vx = kNoMax;            // the largest score, the largest contribution
        auto top = [&](const uint32_t* s, float f0, float f1, uint32_t l0, uint32_t l1) {
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const uint32_t* z = s + 16 * g;
            float u = max3(z[0], z[1], z[2]), w = max3(z[3], z[4], z[5]);
            u = max3(u, z[6], z[7]);
            w = max3(w, z[8], z[9]);
            u = max3(u, z[10], z[11]);
            w = max3(w, z[12], z[13]);
            u = max3(u, z[14], z[15]);
            u = fmaxf(u, w) * (g ? f1 : f0);
            mx = fmaxf(mx, u);
            vx = fmaxf(vx, u + __uint_as_float(g ? l1 : l0));
          }
        };
        tmem_wait_ld();
        tmem_ld_32x32b_x32(tH + 32, s1);
        top(s0, kf[0], kf[1], lv.x, lv.y);
        tmem_wait_ld();
        top(s1, kf[2], kf[3], lv.z, lv.w);
        // ---- raise the maxima, and bring O along (its products must be done)
        if (__any_sync(0xffffffffu, mx > m + kRaise || vx > v + kRaise)) {
          const float m2 = fmaxf(m, mx), v2 = fmaxf(fmaxf(v, vx), m2 - kLow);
          const float by = exp2_fast(v - v2);
          l *= exp2_fast(m - m2);
          m = m2;
          v = v2;
          unit = exp2_fast(m - v + kUnit);
          if (u > 2 * k.t0) {
            // the step before's (that these scores are there says that those before it are done, so this
            // barrier is at most one phase behind: a wait cannot tell more)
            TILE_WAIT(bar.o_done[w][h ^ 1], ((it - 1) >> 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 8; c++) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(tO + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * by);
              tmem_st_32x32b_x16(tO + 16 * c, o);
            }
          }
        }
        // ---- weights: p = 2^(score - m); the row sum keeps p, the product gets p s_v unit in fp16, over the
        // scores that they came from. (A page that this row does not see may make the factor infinite: its p are 0.)
        const uint64_t nm = two(-m, -m);
        uint64_t l2[2] = {0ull, 0ull};
        uint32_t p[32];
        auto weigh = [&](const uint32_t* s, uint32_t* to, float f0, float f1, float w0, float w1) {
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float fg = g ? f1 : f0, wg = fminf((g ? w1 : w0) * unit, FLT_MAX);
            const uint64_t fg2 = two(fg, fg), wg2 = two(wg, wg);
#pragma unroll
            for (int y = 0; y < 8; y++) {
              const int x = 16 * g + 2 * y;
              const uint64_t z = fma2(two(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), fg2, nm);
              const uint64_t e = two(exp2_fast(lo_of(z)), exp2_fast(hi_of(z)));
              l2[y & 1] = add2(l2[y & 1], e);
              const uint64_t q = mul2(e, wg2);
              to[8 * g + y] = pack2(lo_of(q), hi_of(q), __half());
            }
          }
        };
        weigh(s0, p, kf[0], kf[1], vf[0], vf[1]);
        weigh(s1, p + 16, kf[2], kf[3], vf[2], vf[3]);
        tmem_st_32x32b_x32(tH, p);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&bar.p_full[w][h]);
        l += (lo_of(l2[0]) + hi_of(l2[0])) + (lo_of(l2[1]) + hi_of(l2[1]));
      }
      // ---- the item's (or the part's) result; the next item's queries come meanwhile
      TILE_WAIT(bar.piece_full[(n + 1) % kPieces], ((n + 1) / kPieces) & 1);
      fetch_q(s_piece[(n + 1) % kPieces]);
      TILE_WAIT(bar.o_done[w][0], ((it - 1) >> 1) & 1);
      TILE_WAIT(bar.o_done[w][1], ((it - 1) >> 1) & 1);
      tc_fence_after();
      const float back = exp2_fast(v - m - kUnit);
      uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + ((size_t)(k.row0 + tok0 + my_tok) * a.H + k.head * G + my_head) * kHd);
      auto store = [&](int c, const float* o, float f) {             // 32 columns of this thread's row
        if (!live) return;
#pragma unroll
        for (int x = 0; x < 4; x++)
          out[4 * c + x] = make_uint4(pack2(o[8 * x] * f, o[8 * x + 1] * f, T()), pack2(o[8 * x + 2] * f, o[8 * x + 3] * f, T()),
                                      pack2(o[8 * x + 4] * f, o[8 * x + 5] * f, T()), pack2(o[8 * x + 6] * f, o[8 * x + 7] * f, T()));
      };
      if (k.whole) {
        const float inv = l == 0.f ? 0.f : back / l;
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          uint32_t s[32];
          tmem_ld_32x32b_x32(tO + 32 * c, s);
          tmem_wait_ld();
          store(c, reinterpret_cast<const float*>(s), inv);
        }
        tc_fence_before();
        TILE_PIECE_DONE(n);
        continue;
      }
      // a part: its O column-major (four columns of a row together), which its own thread of the joining
      // CTA reads back the same way
      const int b0 = k.b0, b1 = k.b1;
      auto part_o = [&](int b) { return reinterpret_cast<float4*>(ta.part_o) + ((size_t)(2 * b + (b == b0)) * 2 + w) * 32 * kRows + r; };
      auto part_ml = [&](int b) { return ta.part_ml + ((size_t)(2 * b + (b == b0)) * 2 + w) * kRows + r; };
#pragma unroll 1
      for (int c = 0; c < 4; c++) {
        uint32_t s[32];
        tmem_ld_32x32b_x32(tO + 32 * c, s);
        tmem_wait_ld();
        float4* po = part_o(blockIdx.x) + 8 * c * kRows;
#pragma unroll
        for (int x = 0; x < 8; x++)
          po[x * kRows] = make_float4(__uint_as_float(s[4 * x]) * back, __uint_as_float(s[4 * x + 1]) * back,
                                      __uint_as_float(s[4 * x + 2]) * back, __uint_as_float(s[4 * x + 3]) * back);
      }
      *part_ml(blockIdx.x) = make_float2(m, l);
      tc_fence_before();
      __threadfence();
      warp_arrive(&bar.wg[w]);
      TILE_WAIT(bar.wg[w], wgp & 1);
      wgp++;
      if (r == 0) {
        s_last[w] = atomicInc(&ta.counters[2 * b0 + w], b1 - b0) == (uint32_t)(b1 - b0);
        s_counted[w][b0 == (int)blockIdx.x] = 1;
        __threadfence();
      }
      warp_arrive(&bar.wg[w]);
      TILE_WAIT(bar.wg[w], wgp & 1);
      wgp++;
      if (s_last[w]) {
        __threadfence();
        float M = kNoMax, L = 0.f;
#pragma unroll 1
        for (int b = b0; b <= b1; b++) M = fmaxf(M, __ldcg(part_ml(b)).x);
#pragma unroll 1
        for (int b = b0; b <= b1; b++) {
          const float2 ml = __ldcg(part_ml(b));
          L = fmaf(ml.y, exp2_fast(ml.x - M), L);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          float o[32];
#pragma unroll
          for (int x = 0; x < 32; x++) o[x] = 0.f;
          float4 u[8];
          auto read = [&](int b) {
#pragma unroll
            for (int x = 0; x < 8; x++) u[x] = __ldcg(part_o(b) + (8 * c + x) * kRows);
          };
          read(b0);
#pragma unroll 1
          for (int b = b0; b <= b1; b++) {
            float4 v[8];
#pragma unroll
            for (int x = 0; x < 8; x++) v[x] = u[x];
            const float f = exp2_fast(__ldcg(part_ml(b)).x - M);
            if (b < b1) read(b + 1);
#pragma unroll
            for (int x = 0; x < 8; x++) {
              o[4 * x] = fmaf(v[x].x, f, o[4 * x]);
              o[4 * x + 1] = fmaf(v[x].y, f, o[4 * x + 1]);
              o[4 * x + 2] = fmaf(v[x].z, f, o[4 * x + 2]);
              o[4 * x + 3] = fmaf(v[x].w, f, o[4 * x + 3]);
            }
          }
          store(c, o, inv);
        }
      }
      TILE_PIECE_DONE(n);
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    // ------------------------------------------------------------------ pages to operands
    // A thread: key row % 16 and 16 dims from 16 c on. Eight lanes have the eight c of two neighbouring rows, four
    // of each: neither their loads (a bank each) nor, swizzled into the two blocks, their stores conflict.
    const int c = lane & 7, row = (4 * (warp - 8) + (lane >> 3)) ^ (c >> 2);
    const uint32_t off = (uint32_t)(c >> 2) * kHalf + row * 128;
    const uint32_t off0 = off + (((2 * (c & 3)) ^ (row & 7)) << 4), off1 = off + (((2 * (c & 3) + 1) ^ (row & 7)) << 4);
    auto fetch = [&](const int8_t* data, uint32_t t, uint4* x) {
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        const int y = s_row[t % kPageRing][g];
        x[g] = make_uint4(0, 0, 0, 0);
        if (y >= 0) x[g] = __ldg(reinterpret_cast<const uint4*>(data + (size_t)(y + row) * kHd) + c);
      }
    };
    const uint32_t negate = a.scale < 0.f ? 0x80008000u : 0u;   // a negative scale goes with the keys
    auto store_k = [&](uint32_t base, const uint4* x) {
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        const uint32_t u[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          v[2 * i] = i8_pair(u[i], 0x4140, T());
          v[2 * i + 1] = i8_pair(u[i], 0x4342, T());
        }
        if (negate)
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] ^= negate;
        sts128(base + off0 + 16 * g * 128, make_uint4(v[0], v[1], v[2], v[3]));
        sts128(base + off1 + 16 * g * 128, make_uint4(v[4], v[5], v[6], v[7]));
      }
    };
    auto store = [&](uint32_t base, const uint4* x) {
#pragma unroll
      for (int g = 0; g < kGroups; g++) {
        const uint32_t u[4] = {x[g].x ^ 0x80808080u, x[g].y ^ 0x80808080u, x[g].z ^ 0x80808080u, x[g].w ^ 0x80808080u};
        const uint4 lo = make_uint4(i8_half2(u[0], 0x4140), i8_half2(u[0], 0x4342), i8_half2(u[1], 0x4140), i8_half2(u[1], 0x4342));
        const uint4 hi = make_uint4(i8_half2(u[2], 0x4140), i8_half2(u[2], 0x4342), i8_half2(u[3], 0x4140), i8_half2(u[3], 0x4342));
        sts128(base + off0 + 16 * g * 128, lo);
        sts128(base + off1 + 16 * g * 128, hi);
      }
    };
    // the tiles of all pieces are one stream: tile t's loads are issued while tile t - 1 is stored
    uint4 x[kGroups], y[kGroups];
#pragma unroll 1
    for (uint32_t nx = 0;; nx++) {
      const uint32_t t = nx - 1, st = t & 1;       // stored here; nothing yet when nx = 0
      TILE_WAIT(bar.page_full[nx % kAhead], (nx / kAhead) & 1);
      const bool more = s_row[nx % kPageRing][0] != -2;
      if (nx > 0) {
        if (t > 1) TILE_WAIT(bar.k_empty[st], ((t >> 1) - 1) & 1);
        store_k(smK + st * kOperand, x);
        fence_async_smem();
        warp_arrive(&bar.k_full[st]);
      }
      if (more) fetch(a.c.k, nx, x);
      if (nx > 0) {
        if (t > 1) TILE_WAIT(bar.v_empty[st], ((t >> 1) - 1) & 1);
        store(smV + st * kOperand, y);
        fence_async_smem();
        warp_arrive(&bar.v_full[st]);
      }
      if (!more) break;
      fetch(a.c.v, nx, y);
      warp_arrive(&bar.page_empty[nx % kAhead]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    if (warp == 13) {
      // ---------------------------------------------------------------- the walk along this CTA's part of the line
      Start p = s_start;
      Span sp = batch.span(p.s);
      int blks = batch.blocks(sp);
      bool quiet = false;
#pragma unroll 1
      for (uint32_t n = 0;; n++) {
        const int slot = n % kPieces;
        // after a wait that ran out it goes on alone, for the parts that the CTA has to count
        if (n >= kPieces && !quiet && !warp_wait(&bar.piece_empty[slot], (n / kPieces - 1) & 1)) {
          quiet = true;
          if (lane == 0) {
            set_status(a.status, UWC_DEV_TIMEOUT);
            s_gave_up = 1;
          }
        }
        Piece& k = s_piece[slot];
        bool end = true;
#pragma unroll 1
        while (p.left > 0 && end) {
          const Item it(a, sp, G, p.blk);
          const int all = kItemCost + it.total, u1 = min(all, p.u0 + p.left);
          if (u1 > kItemCost) {                    // some of its tiles, not only its own cost
            end = false;
            const int rows = min(2 * kRows, sp.n * G - 2 * kRows * p.blk);
            const bool whole = p.u0 <= kItemCost && u1 == all;
            // the CTAs before this one hold the item's tiles before t0, those after it the rest, `per` each
            const int b0 = blockIdx.x - (p.u0 > kItemCost ? (uint32_t)(p.u0 - kItemCost - 1) / (uint32_t)p.per + 1 : 0);
            const int b1 = blockIdx.x + (all > u1 ? (uint32_t)(all - u1 - 1) / (uint32_t)p.per + 1 : 0);
            if (lane == 0 && !whole) s_part[b0 == (int)blockIdx.x] = make_int3(rows, b0, b1);
            if (lane == 0 && !quiet) {
              k.first = 2 * kRows * p.blk;
              k.rows = rows;
              k.row0 = sp.row0;
              k.seq = p.s;
              k.head = p.h;
              k.start = sp.idle ? -1 : sp.start;
              k.t0 = max(p.u0 - kItemCost, 0);
              k.t1 = u1 - kItemCost;
              k.whole = whole;
              k.b0 = b0;
              k.b1 = b1;
              k.lo = it.lo;
              k.hi = it.hi;
              k.sink_end = it.sink_end;
              k.tA = it.tA;
              k.tB0 = it.tB0;
            }
          }
          p.left -= u1 - p.u0;
          p.u0 = 0;
          if (p.left > 0 && ++p.blk == blks) {
            p.blk = 0;
            if (++p.h == Hkv) {
              p.h = 0;
              do {
                sp = batch.span(++p.s);
                blks = batch.blocks(sp);
              } while (blks == 0 && p.s + 1 < a.b.seqs);
            }
          }
        }
        if (end && !quiet && lane == 0) k.rows = 0;
        __syncwarp();
        if (lane == 0 && !quiet) mbar_arrive(&bar.piece_full[slot]);
        if (end) break;
      }
    } else if (warp == 14 && (ta.withhold & blockIdx.x & 1)) {
      // the hook: no tile is handed over
    } else if (warp == 14) {
      // ---------------------------------------------------------------- the pages: a lane a 16-key group, four tiles at once
      const int grp = lane & (kGroups - 1);
      const float qmul = fabsf(a.scale) * kLog2OfE;
      uint32_t t = 0;
#pragma unroll 1
      for (uint32_t n = 0;; n++) {
        TILE_PIECE(n);
        auto look = [&](int i0, int& y, float2& sc) {
          const int i = i0 + lane / kGroups, j = k.key(i) + 16 * grp;
          y = -1;
          sc = make_float2(kNoScore, 0.f);
          if (i < k.t1 && k.seen(j, 16)) {
            const int page = page_at(a.b, a.c, k.seq, j >> a.c.lg);
            if (page < 0) {
              set_status(a.status, UWC_DEV_RANGE);
            } else {
              const int ph = page * Hkv + k.head;      // rows of the pool fit an int: the host checks
              y = ph * ps + (j & (ps - 1));
              sc = make_float2(fmaxf(__ldg(a.c.sk + ph) * qmul, kNoScore), __ldg(a.c.sv + ph));
            }
          }
        };
        int y = -1, ny;
        float2 sc = make_float2(kNoScore, 0.f), nsc;
        // the look-up of four tiles ahead of their hand-over
#pragma unroll 1
        for (int i0 = k.t0 - kAhead; i0 < k.t1; i0 += kAhead) {
          look(i0 + kAhead, ny, nsc);
#pragma unroll 1
          for (int i = 0; i < kAhead && i0 >= k.t0 && i0 + i < k.t1; i++, t++) {
            if (t >= kAhead) TILE_WAIT(bar.page_empty[t % kAhead], (t / kAhead - 1) & 1);
            const unsigned unseen = __ballot_sync(0xffffffffu, y < 0) >> (i * kGroups) & ((1u << kGroups) - 1);
            if (lane / kGroups == i) {
              s_row[t % kPageRing][grp] = y;
              s_scale[t % kPageRing][grp] = sc;
              s_log[t % kPageRing][grp] = __log2f(fabsf(sc.y));
              if (grp == 0) s_unseen[t % kPageRing] = (int)unseen;
            }
            warp_arrive(&bar.page_full[t % kAhead]);
          }
          y = ny;
          sc = nsc;
        }
        TILE_PIECE_DONE(n);
      }
      if (t >= kAhead) TILE_WAIT(bar.page_empty[t % kAhead], (t / kAhead - 1) & 1);
      if (lane == 0) {
        s_row[t % kPageRing][0] = -2;
        mbar_arrive(&bar.page_full[t % kAhead]);
      }
    } else {
      // ------------------------------------------------------------------ the products of a row tile
      const int w = warp == 15;
      const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128, smq = smQ + w * kOperand;
      uint32_t it = 0, own = 0, items = 0;         // tiles; this row tile's tiles and items (its barriers' phases)
      auto scores = [&](uint32_t st, uint32_t h) { // 64 keys
        const uint32_t kk = smK + st * kOperand + h * 64 * 128;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const uint32_t off = (x >> 2) * kHalf + (x & 3) * 32;
          mma_ss(tS + 64 * h, sdesc_sw128(smq + off), sdesc_sw128(kk + off), kIdescS | IsBf16<T>::value * ((1u << 7) | (1u << 10)), x > 0);
        }
        mbar_arrive(&bar.s_full[w][h]);
        mma_commit(&bar.s_full[w][h]);
      };
      auto outputs = [&](uint32_t st, uint32_t h, uint32_t acc) {
        const uint32_t v = smV + st * kOperand + h * 8192;
#pragma unroll
        for (int x = 0; x < 4; x++) mma_ts(tO, tS + 64 * h + 8 * x, sdesc_mn(v + x * 2048), kIdescO, acc || x > 0);
        mma_commit(&bar.o_done[w][h]);
      };
#pragma unroll 1
      for (uint32_t n = 0;; n++) {
        TILE_PIECE(n);
        const bool mine = k.rows > kRows * w;
        const int T1 = k.t1 - k.t0;
        TILE_PIECE_DONE(n);
        if (!mine) {                               // no rows: this warp's word that the stages are free
#pragma unroll 1
          for (int j = 0; j < T1; j++, it++) {
            TILE_WAIT(bar.k_full[it & 1], (it >> 1) & 1);
            warp_arrive(&bar.k_empty[it & 1]);
            TILE_WAIT(bar.v_full[it & 1], (it >> 1) & 1);
            warp_arrive(&bar.v_empty[it & 1]);
          }
          continue;
        }
        // the first tile's scores
        TILE_WAIT(bar.k_full[it & 1], (it >> 1) & 1);
        TILE_WAIT(bar.q_full[w], items & 1);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll 1
          for (uint32_t h = 0; h < 2; h++) scores(it & 1, h);
          mma_commit(&bar.k_empty[it & 1]);
        }
        __syncwarp();
        items++;
#pragma unroll 1
        for (int j = 0; j < T1; j++, it++, own++) {
          const uint32_t st = it & 1, nx = it + 1;
          const bool more = j + 1 < T1;
          TILE_WAIT(bar.v_full[st], (it >> 1) & 1);
          if (more) TILE_WAIT(bar.k_full[nx & 1], (nx >> 1) & 1);
#pragma unroll 1
          for (uint32_t h = 0; h < 2; h++) {
            TILE_WAIT(bar.p_full[w][h], own & 1);
            tc_fence_after();
            if (elect_one()) {
              outputs(st, h, j > 0 || h > 0);
              if (h) mma_commit(&bar.v_empty[st]);
              if (more) {
                scores(nx & 1, h);
                if (h) mma_commit(&bar.k_empty[nx & 1]);
              }
            }
            __syncwarp();
          }
        }
      }
    }
  }
  if (false) {
  timeout:
    if (lane == 0) {
      set_status(a.status, UWC_DEV_TIMEOUT);
      s_gave_up = 1;
    }
  }
  __syncwarp();
  if (warp == 12 || warp == 15) {
    // every product that was issued has landed before the tensor memory goes (bounded, as every wait)
    if (elect_one()) mma_commit(&bar.fin);
    __syncwarp();
  }
  if (warp == 12) {
#pragma unroll 1
    for (int n = 0; n < (1 << 20) && !mbar_try_wait(&bar.fin, 0); n++) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
    // parts that a wait which ran out left uncounted: their items' counters end at zero all the same, for the next
    // call with this workspace (this one's rows are lost, as the status says)
    if (s_gave_up && lane == 0)
#pragma unroll 1
      for (int i = 0; i < 4; i++)
        if (s_part[i & 1].x > kRows * (i >> 1) && !s_counted[i >> 1][i & 1])
          atomicInc(&ta.counters[2 * s_part[i & 1].y + (i >> 1)], s_part[i & 1].z - s_part[i & 1].y);
  }
}

int tile_grid(int seqs, int max_new, int max_len, int H, int Hkv, int window, int sinks) {
  long long keys = max_len;
  if (window >= 0) keys = std::min(keys, (long long)window + max_new + 3ll * kTile + std::min(sinks, max_len));
  const long long blocks = ((long long)max_new * (H / Hkv) + 2 * kRows - 1) / (2 * kRows);
  const long long tiles = std::max(1ll, (keys + kTile - 1) / kTile);
  const double all = (double)blocks * tiles * seqs * Hkv;
  return (int)std::max(1.0, std::min((double)std::min(uwc_num_sms(), 512), all));
}

constexpr uint64_t kCounterBytes = 4096;

}  // namespace

uint64_t uwc_paged_tile_workspace(int seqs, int max_new, int max_len, int H, int Hkv, int window, int sinks) {
  const uint64_t grid = tile_grid(seqs, max_new, max_len, H, Hkv, window, sinks);
  return kCounterBytes + grid * 2 * 2 * kRows * (kHd * 4 + 8);
}

int uwc_paged_tile_launch(const AttnArgs* a, int dtype, int max_len, void* workspace, cudaStream_t stream) {
  const int grid = tile_grid(a->b.seqs, a->b.max_new, max_len, a->H, a->c.Hkv, a->window, a->sinks);
  TileArgs ta;
  ta.a = *a;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ta.counters = reinterpret_cast<uint32_t*>(ws);
  ta.part_o = reinterpret_cast<float*>(ws + kCounterBytes);
  ta.part_ml = reinterpret_cast<float2*>(ta.part_o + (size_t)grid * 4 * kRows * kHd);
  ta.withhold = uwc_withhold();
  const void* fn = dtype == UWC_T_BF16 ? (const void*)k_paged_tile<__nv_bfloat16> : (const void*)k_paged_tile<__half>;
  const int rc = uwc_paged_allow_smem(fn, kSmem);
  if (rc != UWC_OK) return rc;
  if (dtype == UWC_T_BF16) k_paged_tile<__nv_bfloat16><<<grid, kThreads, kSmem, stream>>>(ta);
  else k_paged_tile<__half><<<grid, kThreads, kSmem, stream>>>(ta);
  uwc_count_launch();
  return uwc_launch_status();
}
