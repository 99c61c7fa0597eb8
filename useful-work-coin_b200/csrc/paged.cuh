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
  const int hi = min(c1, b.rows);
  r.n = min(max(hi - r.row0, 0), b.max_new);
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

}  // namespace paged

// The checks that every paged call shares (paged.cu).
int uwc_paged_check(const paged::Cache* cache, const paged::Seqs* seqs);
