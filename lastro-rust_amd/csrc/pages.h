// The paged 16-bit K/V cache of include/moert.h (moert_pages_*): device view, index arithmetic and launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dev_math.h"
#include "kv8.h"

namespace moert {

constexpr int kPgBlock = 32;  // positions of a block of K or V within a page
enum { PG_ROWS = 0, PG_REFUSED = 1, PG_FROM = 2, PG_STATE = 4 };  // words of a sequence's state

struct PagesDev {
  int seqs, kvh, d, pages, max_pages;
  int lp;  // log2 of a page's positions
  int bf16;
  uint16_t *k, *v;
  int *table, *state, *free;
};

// Place of position t, element e in a block: K as the columns of a product take it, 8 elements of a row at a time; V as
// the rows of the second product do, the 8 positions of an element that one lane of the first product holds.
__host__ __device__ __forceinline__ constexpr int pg_k_place(int t, int e) { return (e / 8 * kPgBlock + t) * 8 + e % 8; }
__host__ __device__ __forceinline__ constexpr int pg_v_place(int d, int t, int e) {
  return ((t / 16 * 2 + t % 8 / 4) * d + e) * 8 + t % 4 + t % 16 / 8 * 4;
}

// Rows of a sequence, whatever the state holds.
__device__ __forceinline__ int pg_rows(const PagesDev& c, int s) {
  const int n = c.state[(size_t)s * PG_STATE + PG_ROWS], most = c.max_pages << c.lp;
  return n < 0 ? 0 : n > most ? most : n;
}
// Rows that its positions see: none of a sequence that the last plan has refused.
__device__ __forceinline__ int pg_seen(const PagesDev& c, int s) {
  return c.state[(size_t)s * PG_STATE + PG_FROM] < 0 ? 0 : pg_rows(c, s);
}
// A page is used as an index only after this: whatever the table holds, it stays inside the pool.
__device__ __forceinline__ int pg_page(const PagesDev& c, int raw) { return (unsigned)raw < (unsigned)c.pages ? raw : 0; }
// The pool's block of a KV head's rows [32 b, 32 b + 32) in a sequence, from its page; below 2^30.
__device__ __forceinline__ int pg_block(const PagesDev& c, int page, int h, int b) {
  const int l = c.lp - 5;
  return ((page * c.kvh + h) << l) + (b & ((1 << l) - 1));
}

// Rows [lo, hi) of a sequence in a packed batch, whatever the starts hold; without starts one of each sequence.
__device__ __forceinline__ int2 pg_span(const int* starts, int s, int tokens) {
  if (!starts) return make_int2(s, s + 1);
  const int lo = min(max(starts[s], 0), tokens), hi = min(max(starts[s + 1], lo), tokens);
  return make_int2(lo, hi);
}

size_t pages_workspace(const PagesDev& c, int heads, int tokens);

hipError_t launch_pages_clear(hipStream_t s, const PagesDev& c);
hipError_t launch_pages_plan(hipStream_t s, const PagesDev& c, const int* fresh, int tokens, int* starts, int* slots,
                             int* positions);
hipError_t launch_pages_append(hipStream_t s, const PagesDev& c, KvRows k, KvRows v, const int* slots, int tokens);
hipError_t launch_pages_attend(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, void* ws, size_t ws_bytes);
hipError_t launch_pages_prompt(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, int least, void* ws, size_t ws_bytes);

}  // namespace moert
