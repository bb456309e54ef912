// Attention over the paged 16-bit K/V cache (pages.h).
#include "pages_dev.h"

namespace moert {

namespace {

template <int BF16>
__device__ __forceinline__ float held_value(uint16_t x) {
  return BF16 ? __uint_as_float((uint32_t)x << 16) : h2f(x);
}
// bf16 bits of a float, to nearest, ties to even; NaN stays.
__device__ __forceinline__ uint16_t f2bf(float x) {
  const uint32_t w = __float_as_uint(x);
  return x != x ? 0x7fff : (uint16_t)((w + 0x7fff + (w >> 16 & 1)) >> 16);
}

// A wave per row and query head, 64 positions at a time: a lane's score is of one position, its output of D / 64
// elements. one: only sequences of one row, otherwise those of at least `least`.
template <int D, int BF16>
__global__ __launch_bounds__(256) void k_pages_rows(PagesDev c, KvRows q, KvRows out, const int* starts, int tokens,
                                                    int heads, float scale, int one, int least) {
  const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= (long long)tokens * heads) return;
  const int lane = threadIdx.x & 63, i = (int)(u / heads), a = (int)(u % heads), h = a / (heads / c.kvh);
  int s = i;
  if (starts) {
    int lo = 0;
    for (int hi = c.seqs; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= i) lo = mid;
      else hi = mid;
    }
    s = lo;
  }
  const int2 span = pg_span(starts, s, tokens);
  const int n = span.y - span.x;
  if (i < span.x || i >= span.y || (one ? n != 1 : n < least)) return;
  const int sees = pg_seen(c, s) - n + 1 + i - span.x;
  float x[D], o[D / 64] = {}, m = -3.4e38f, l = 0.0f;
  const long long qa = i * q.pos + a * q.head;
  for (int e = 0; e < D; e++)
    x[e] = q.f16 ? held_value<BF16>(((const uint16_t*)q.p)[qa + e]) : ((const float*)q.p)[qa + e];
  for (int t0 = 0; t0 < sees; t0 += 64) {
    const int t = min(t0 + lane, sees - 1);
    const int page = pg_page(c, c.table[(size_t)s * c.max_pages + (t >> c.lp)]);
    const size_t at = (size_t)pg_block(c, page, h, t / kPgBlock) * (kPgBlock * D);
    float sc = 0.0f;
    for (int e = 0; e < D; e++) sc = fmaf(x[e], held_value<BF16>(c.k[at + pg_k_place(t % kPgBlock, e)]), sc);
    sc *= scale;
    if (t0 + lane >= sees) sc = -3.4e38f;
    const float mn = fmaxf(m, group_max(sc)), al = expf(m - mn);
    const float p = t0 + lane < sees ? expf(sc - mn) : 0.0f;
    m = mn;
    l = l * al + group_sum(p);
    for (int j = 0; j < D / 64; j++) o[j] *= al;
    for (int y = 0; y < 64 && t0 + y < sees; y++) {
      const int ty = t0 + y, pgy = pg_page(c, c.table[(size_t)s * c.max_pages + (ty >> c.lp)]);
      const size_t ay = (size_t)pg_block(c, pgy, h, ty / kPgBlock) * (kPgBlock * D);
      const float py = __shfl(p, y);
      for (int j = 0; j < D / 64; j++)
        o[j] = fmaf(py, held_value<BF16>(c.v[ay + pg_v_place(D, ty % kPgBlock, lane + 64 * j)]), o[j]);
    }
  }
  const long long oa = i * out.pos + a * out.head + lane;
  for (int j = 0; j < D / 64; j++) {
    const float y = sees > 0 ? o[j] / l : 0.0f;
    if (out.f16) ((uint16_t*)out.p)[oa + 64 * j] = BF16 ? f2bf(y) : f2h(y);
    else ((float*)out.p)[oa + 64 * j] = y;
  }
}

hipError_t rows_of(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out, const int* starts,
                   int tokens, int one, int least) {
  const unsigned grid = (unsigned)(((long long)tokens * heads + 3) / 4);
#define ROWS(DD, BB) \
  if (c.d == DD && c.bf16 == BB) klaunch(k_pages_rows<DD, BB>, grid, 256, 0, s, c, q, out, starts, tokens, heads, scale, one, least);
  ROWS(64, 0) ROWS(64, 1) ROWS(128, 0) ROWS(128, 1)
#undef ROWS
  return hipGetLastError();
}

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

}  // namespace

size_t pages_workspace(const PagesDev& c, int heads, int tokens) { return 0; }

hipError_t launch_pages_attend(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, void* ws) {
  return rows_of(s, c, heads, scale, q, out, starts, tokens, 1, 1);
}

hipError_t launch_pages_prompt(hipStream_t s, const PagesDev& c, int heads, float scale, KvRows q, KvRows out,
                               const int* starts, int tokens, int least, void* ws) {
  return launch_pages_tiles(s, args(c, heads, scale, q, out, starts, tokens, least, 1 << 30));
}

}  // namespace moert
