// How an attention over the paged 16-bit K/V cache goes about its work (pages.h): which kernel, how many splits.
#include "pages_dev.h"

namespace moert {

namespace {

PgArgs args(const PagesDev& c, int heads, float scale, KvRows q, KvRows out, const int* starts, int tokens, int least,
            int most) {
  PgArgs a{};
  a.c = c, a.q = q, a.out = out, a.starts = starts;
  a.tokens = tokens, a.g = heads / c.kvh;
  a.least = least, a.most = most;
  a.vec = wide_rows(q) | wide_rows(out) << 1;
  a.kf = frexpf(__builtin_fabsf(scale), &a.ke) * kPgLog2e;
  a.sign = scale < 0.0f ? 0x80000000u : 0u;
  return a;
}

// Splits cost a second launch and the partials' way through memory, about what a wave takes for 7 blocks: none where a wave
// of a full table keeps at most 24 (1000 of 1280 positions, 8 KV heads: 8.6 us without, 10.9 with 3; sixteen sequences of up
// to 2000 of 2560: 13.7 without, 15.9 with 2; 4097 of 4608: 24.1 without, 11.5 with 12). Then one workgroup for each of 256
// compute units, and more (up to 1024, four to a unit) only while a wave keeps 16 blocks; never fewer than 3 a wave. (131000
// positions, 8 KV heads: 43.1 us with 64 splits, 44.1 with 32, 50.6 with 16.)
int cols_splits(const PagesDev& c, long long units) {
  const int blocks = c.max_pages << (c.lp - 5), cap = blocks / 12, most = cap > kPgMaxSplits ? kPgMaxSplits : cap;
  if (blocks <= 24 * 4) return 1;
  long long s = 256 / units > 1 ? 256 / units : 1;
  while (2 * s * units <= 1024 && blocks / (8 * s) >= 16) s *= 2;
  return (int)(s < most ? s : most);
}

constexpr int kTilesAtOnce = 512;

// Tiles of 128 rows, where there are fewer than two workgroups to a unit: splits, of at least 16 blocks of a full table
// each. (64 positions after 16000, 8 KV heads of 128: 407 us without splits, 59, 47 and 42 with 256, 512 and 768 workgroups
// at most; 16 sequences of up to 100 after 500, 3 query heads each: 19.5 us without, 19.8 with 512, 26.7 with 768.)
int tiles_splits(const PagesDev& c, long long units) {
  const int blocks = c.max_pages << (c.lp - 5), cap = blocks / 16;
  const int most = cap < 1 ? 1 : cap > kPgMaxSplits ? kPgMaxSplits : cap;
  const long long s = kTilesAtOnce / units;
  return (int)(s < 1 ? 1 : s < most ? s : most);
}

// Whether the tiles of 16 rows that the waves of a workgroup share do better than those of 128 rows that they split: up to
// 48 rows of a sequence on average, of wide heads 32. (8 KV heads of 64, 48 rows: 4000 positions 11.4 us in the one, 14.1 in
// the other, 32000 25.5 and 21.7, of eight sequences of 4000 17.5 and 23.4; of 128, 32 rows: 12.4 and 18.8, 33.5 and 30.5,
// 25.5 and 30.3, but 44 rows of 64 sequences of 1000 59.3 and 42.5.) The average is all that the host knows, and the rule
// holds for what is like it: after long texts 128 rows would do better (the two figures at 32000), and where one sequence
// has the rows and most have few or none, it runs as one of few rows does. (3 heads of 64 in fp16, 4 of 128 in bf16; the
// sequence's rows in 128 and beside other sequences' single rows in 16: 300 rows beside 63 8.7 and 6.8 us, 12.1 and 14.8;
// 900, 440 of wide heads, 16.1 and 18.9, 15.0 and 21.7; 300 after 16000 59 and 105, 113 and 337; 5000 beside 999 106 and
// 280, 218 and 819.) A caller who knows of one calls for it alone.
bool few_rows(const PgArgs& a) { return (long long)a.tokens * a.g <= (a.c.d == 64 ? 48ll : 32ll) * a.c.seqs; }

size_t up(size_t x) { return (x + 255) / 256 * 256; }
size_t share_bytes(const PagesDev& c, size_t rows) { return up(rows * 8) + up(rows * c.d * 4); }

// Whether the workspace does for the splits; where it lies for them.
bool place(PgArgs* a, void* ws, size_t bytes, int width) {
  if (a->splits == 1) return true;
  const size_t rows = (size_t)a->tiles * a->c.kvh * width * a->splits;
  a->ml = (float2*)ws;
  a->part = (float*)((char*)ws + up(rows * 8));
  return share_bytes(a->c, rows) <= bytes;
}

}  // namespace

size_t pages_workspace(const PagesDev& c, int heads, int tokens) {
  const int g = heads / c.kvh, tiles = c.seqs * ((g + 15) / 16), splits = cols_splits(c, (long long)tiles * c.kvh);
  size_t rows = splits > 1 ? (size_t)tiles * c.kvh * 16 * splits : 0;
  if (tokens) {  // of as many rows and of fewer: never less than for fewer
    const size_t most = (size_t)(c.max_pages << (c.lp - 5)) / 8 < kPgMaxSplits ? (c.max_pages << (c.lp - 5)) / 8 : kPgMaxSplits;
    const size_t few = ((size_t)tokens * g / 16 + c.seqs) * c.kvh, many = ((size_t)tokens * g / 128 + c.seqs) * c.kvh;
    const size_t a = few * most < 1024 ? few * most : 1024, b = many * most < kTilesAtOnce ? many * most : kTilesAtOnce;
    if (most > 1 && rows < a * 16) rows = a * 16;
    if (most > 1 && rows < b * 128) rows = b * 128;
  }
  return rows ? share_bytes(c, rows) : 0;
}

hipError_t launch_pages_attend(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, void* ws, size_t ws_bytes) {
  PgArgs a = args(c, heads, scale, q, out, starts, tokens, 1, 1);
  a.tiles = pg_tiles(a, 16);
  a.splits = cols_splits(c, (long long)a.tiles * c.kvh);
  if (!place(&a, ws, ws_bytes, 16)) return hipErrorInvalidValue;
  if (const hipError_t e = launch_pages_cols(s, a)) return e;
  return a.splits > 1 ? launch_pages_join(s, a, 16) : hipSuccess;
}

hipError_t launch_pages_prompt(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, int least, void* ws, size_t ws_bytes) {
  PgArgs a = args(c, heads, scale, q, out, starts, tokens, least, 1 << 30);
  const int width = few_rows(a) ? 16 : 128;
  a.tiles = pg_tiles(a, width);
  const long long units = (long long)a.tiles * c.kvh;
  a.splits = width == 16 ? cols_splits(c, units) : tiles_splits(c, units);
  if (!place(&a, ws, ws_bytes, width)) return hipErrorInvalidValue;
  if (const hipError_t e = width == 16 ? launch_pages_cols(s, a) : launch_pages_tiles(s, a)) return e;
  return a.splits > 1 ? launch_pages_join(s, a, width) : hipSuccess;
}

}  // namespace moert
