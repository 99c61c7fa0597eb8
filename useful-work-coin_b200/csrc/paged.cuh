// What the paged-cache kernels share: the cache and the ragged batch as the kernels see them.
//
// A cache is a pool of pages of one layer: keys and values (pages, Hkv, page_size, 128) int8 and one
// float32 scale for each (page, KV head), so a value is its integer times its page's scale. A batch
// is ragged: rows cu[s] .. cu[s + 1] - 1 are sequence s's new tokens, at positions start[s] and on;
// row s of the table lists the sequence's pages. All of it is read on the device (one CUDA graph
// serves every step), so every index is checked there before it is used: what is out of range is
// skipped and raises UWC_DEV_RANGE.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "uwc_device.cuh"

namespace paged {

constexpr int kHd = 128;   // head dimension

struct Cache {
  int8_t* k;
  float* sk;
  int8_t* v;
  float* sv;
  int pages, ps, Hkv;
  int lg;                  // log2 of ps
};

struct Seqs {
  const int* table;        // (seqs, width)
  const int* start;        // position of the first new token; negative: an idle slot
  const int* cu;           // seqs + 1 row offsets
  int seqs, width, rows;   // rows: rows of the row tensors (every row index is below it)
  int max_new;             // at least every sequence's new tokens
};

// One sequence's new tokens: rows row0 .. row0 + n - 1 at positions start .. start + n - 1.
struct Span {
  int row0, n, start;
  bool idle;               // the slot is idle (start < 0): its rows are there, its pages are not
  bool bad;                // the metadata was out of range; n is what of it is in range
};

__device__ __forceinline__ Span span_of(const Seqs& b, int ps, int s) {
  const int c0 = __ldg(b.cu + s), c1 = __ldg(b.cu + s + 1);
  Span r;
  r.start = __ldg(b.start + s);
  r.row0 = max(c0, 0);
  r.idle = r.start < 0;
  const int hi = max(min(c1, b.rows), r.row0);     // no difference below overflows, whatever the two hold
  r.n = min(hi - r.row0, b.max_new);
  if (!r.idle) r.n = max(0, min(r.n, b.width * ps - r.start));   // width * ps < 2^31: the host checks
  r.bad = c0 < 0 || c1 < c0 || r.n != c1 - c0;
  return r;
}

// Page of a sequence's position, -1 where the table has none.
__device__ __forceinline__ int page_at(const Seqs& b, const Cache& c, int s, int slot) {
  if (slot < 0 || slot >= b.width) return -1;
  const int id = __ldg(b.table + (size_t)s * b.width + slot);
  return id >= 0 && id < c.pages ? id : -1;
}

// ---- attention
struct AttnArgs {
  Cache c;
  Seqs b;
  const void* q;           // element (n, h, d) at n * q_tok + h * q_head + d
  long long q_tok, q_head;
  void* out;               // (rows, H, 128)
  int H, window, sinks;    // window < 0: none
  float scale;
  uint32_t* status;
};

// The keys that tokens t0 .. t1 of a sequence see, as tiles of TILE keys: tiles 0 .. tA - 1 hold the
// sinks, then tB0 .. on the windows. There is at least one tile, seen or not: it writes the zeros.
template <int TILE>
struct Keys {
  int p0, p1;              // positions of the first and the last row
  int lo, hi, sink_end;    // windows: keys lo .. hi - 1; sinks: keys below sink_end
  int tA, tB0, total;
  __device__ __forceinline__ Keys(const AttnArgs& a, const Span& sp, int t0, int t1) {
    p0 = sp.idle ? -1 : sp.start + t0;
    p1 = sp.idle ? -1 : sp.start + t1;
    hi = a.window == 0 ? 0 : p1 + 1;
    lo = a.window < 0 ? 0 : max(0, p0 - a.window + 1);
    sink_end = a.window < 0 ? 0 : min(a.sinks, p1 + 1);
    tA = (sink_end + TILE - 1) / TILE;
    tB0 = max(tA, lo / TILE);
    total = max(1, tA + max(0, (hi + TILE - 1) / TILE - tB0));
  }
  // the first key of tile i
  __device__ __forceinline__ int key(int i) const { return (i < tA ? i : tB0 + (i - tA)) * TILE; }
  // whether some row sees one of the n keys from j on
  __device__ __forceinline__ bool seen(int j, int n) const { return j < sink_end || (j < hi && j + n > lo); }
  // whether every row sees all of them
  __device__ __forceinline__ bool full(const AttnArgs& a, int j, int n) const {
    return j + n - 1 <= p0 && (a.window < 0 || j > p1 - a.window || j + n <= a.sinks);
  }
};
__device__ __forceinline__ bool sees(const AttnArgs& a, int pos, int j) {
  return j <= pos && (a.window < 0 || j > pos - a.window || j < a.sinks);
}

// Two 16-bit values as float32, and back.
__device__ __forceinline__ float2 two_f(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 two_f(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two of four int8 values as an fp16 pair, exactly: with the values biased by 128 (the caller's
// xor 0x80), 0x6400 | byte is the fp16 number 1024 + byte. sel 0x4140: bytes 0, 1; 0x4342: bytes 2, 3.
__device__ __forceinline__ uint32_t i8_half2(uint32_t biased, uint32_t sel) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, sel), k = 0x64806480u;   // 1152, twice
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The exponent e that brings a row whose largest magnitude is mx to [2^14, 2^15) (up to 2^127, down to 2^-86; what is
// smaller still stays below that): q 2^e is its fp16 form.
__device__ __forceinline__ int row_exponent(float mx) {
  const int x = (__float_as_int(mx) >> 23) & 255;
  return mx == 0.f || x == 255 ? 0 : min(14 + 127 - x, 100);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// A wait of a whole warp in few instructions (a kernel of many roles lives on its instruction cache): up to
// 2^18 polls, each of which the hardware suspends for about 4 us while the barrier is not ready, so about a second
// (2^23 of them took 35). The same answer in all lanes: false when it ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  uint32_t left = 1u << 18;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "POLL_%=:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE_%=;\n\t"
      "sub.u32 %0, %0, 1;\n\t"
      "setp.ne.u32 p, %0, 0;\n\t"
      "@p bra POLL_%=;\n\t"
      "DONE_%=:\n\t}"
      : "+r"(left)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, left != 0);
}
// One arrival for a warp, after all that its lanes did before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

constexpr float kNoMax = -1e30f;             // a running maximum before any key
constexpr float kLog2OfE = 1.4426950408889634f;

}  // namespace paged

// The form of uwc_paged_attention for more rows than the few-row form takes (paged_tile.cu).
uint64_t uwc_paged_tile_workspace(int seqs, int max_new, int max_len, int H, int Hkv, int window, int sinks);
int uwc_paged_tile_launch(const paged::AttnArgs* a, int dtype, int max_len, void* workspace, cudaStream_t stream);

// Dynamic shared memory beyond 48 KiB, asked for once per kernel and device (paged_attn.cu).
int uwc_paged_allow_smem(const void* kernel, int bytes);

// The checks that every paged call shares; sets cache->lg (paged.cu).
int uwc_paged_check(paged::Cache* cache, const paged::Seqs* seqs);
