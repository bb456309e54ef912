// How an attention over the paged 16-bit K/V cache goes about its work (pages.h): which kernel, how many splits.
#include "pages_dev.h"

namespace moert {

namespace {

PgArgs args(const PagesDev& c, int heads, float scale, KvRows q, KvRows out, const int* starts, int tokens, int least,
            int most) {
  PgArgs a{};
  a.c = c, a.q = q, a.out = out, a.starts = starts;
  a.tokens = tokens, a.heads = heads, a.g = heads / c.kvh;
  a.least = least, a.most = most;
  a.vec = wide_rows(q) | wide_rows(out) << 1;
  a.kf = frexpf(__builtin_fabsf(scale), &a.ke) * kPgLog2e;
  a.sign = scale < 0.0f ? 0x80000000u : 0u;
  return a;
}

// Splits cost a second launch and the partials' way through memory: one workgroup for each of 256 compute units, and more
// (up to 1024, four to a unit) only while a wave keeps 16 blocks of a full table; never fewer than 3 a wave.
int cols_splits(const PagesDev& c, long long units) {
  const int blocks = c.max_pages << (c.lp - 5), cap = blocks / 12;
  const int most = cap < 1 ? 1 : cap > kPgMaxSplits ? kPgMaxSplits : cap;
  long long s = 256 / units > 1 ? 256 / units : 1;
  while (2 * s * units <= 1024 && blocks / (8 * s) >= 16) s *= 2;
  return (int)(s < most ? s : most);
}

size_t up(size_t x) { return (x + 255) / 256 * 256; }
size_t share_bytes(const PagesDev& c, size_t rows) { return up(rows * 8) + up(rows * c.d * 4); }

void place(PgArgs* a, void* ws, int width) {
  if (a->splits == 1) return;
  a->ml = (float2*)ws;
  a->part = (float*)((char*)ws + up((size_t)a->tiles * a->c.kvh * width * a->splits * 8));
}

}  // namespace

size_t pages_workspace(const PagesDev& c, int heads, int tokens) {
  const int tiles = c.seqs * ((heads / c.kvh + 15) / 16), splits = cols_splits(c, (long long)tiles * c.kvh);
  return splits > 1 ? share_bytes(c, (size_t)tiles * c.kvh * 16 * splits) : 0;
}

hipError_t launch_pages_attend(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, void* ws) {
  PgArgs a = args(c, heads, scale, q, out, starts, tokens, 1, 1);
  a.tiles = pg_tiles(a, 16);
  a.splits = cols_splits(c, (long long)a.tiles * c.kvh);
  place(&a, ws, 16);
  if (const hipError_t e = launch_pages_cols(s, a)) return e;
  return a.splits > 1 ? launch_pages_join(s, a, 16) : hipSuccess;
}

hipError_t launch_pages_prompt(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, int least, void* ws) {
  PgArgs a = args(c, heads, scale, q, out, starts, tokens, least, 1 << 30);
  a.tiles = pg_tiles(a, 128);
  a.splits = 1;
  return launch_pages_tiles(s, a);
}

}  // namespace moert
