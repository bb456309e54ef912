// The paged 16-bit K/V cache: planning a step's pages, appending rows, and the C entry points (pages_attn.hip has the
// attention).
#include "pages.h"

#include "../../include/moert.h"
#include "launch.h"
#include "rows_api.h"

namespace moert {

namespace {

__global__ __launch_bounds__(256) void k_pages_clear(PagesDev c) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < c.seqs * PG_STATE) c.state[i] = 0;
  if (i == 0) c.free[0] = c.pages;
  if (i < c.pages) c.free[1 + i] = c.pages - 1 - i;  // the last is given first
}

// Sums over the threads before this one and over all of them, none above `most` (of terms in [0, most], most < 2^30). lds:
// no other scan's.
template <int N>
__device__ __forceinline__ int2 plan_scan(int x, int most, int* lds) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(sum, d);
    if (lane >= d) sum = min(sum + y, most);
  }
  if (lane == 63) lds[w] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < N / 64; i++) {
    if (i == w) before = all;
    all = min(all + lds[i], most);
  }
  const int up = __shfl_up(sum, 1);
  return make_int2(min(before + (lane ? up : 0), most), all);
}

// For each of R numbers the last i in [0, n) with at[i] <= x (at[0] <= x, at not falling), side by side.
template <int R>
__device__ __forceinline__ void last_from(const int* at, int n, const int* x, int* lo) {
#pragma unroll
  for (int r = 0; r < R; r++) lo[r] = 0;
  for (int len = n; len > 1;) {
    const int half = len >> 1;
#pragma unroll
    for (int r = 0; r < R; r++) lo[r] += at[lo[r] + half] <= x[r] ? half : 0;
    len -= half;
  }
}

// Slot and position of row i of the batch, row i - start of sequence s.
__device__ __forceinline__ void plan_row(const PagesDev& c, int s, int start, int i, int* slots, int* positions) {
  const int from = c.state[(size_t)s * PG_STATE + PG_FROM], pos = from < 0 ? -1 : from + i - start;
  int slot = -1;
  if (pos >= 0) {
    const int page = c.table[(size_t)s * c.max_pages + min(pos >> c.lp, c.max_pages - 1)];
    if ((unsigned)page < (unsigned)c.pages) slot = (page << c.lp) + (pos & ((1 << c.lp) - 1));
  }
  slots[i] = slot;
  if (positions) positions[i] = pos;
}

constexpr int kRuns = 4;  // pages that a thread moves side by side: each waits for a search and two accesses

// One workgroup of N threads takes the sequences N at a time: sums over them, in order, say where the pages of each lie on
// the free stack, and all threads together move the pages. With `place` (N sequences at most) also the rows' slots. Bound
// by latency: what a thread looks up one after the other. 64 sequences of a row each in 4.7 us, 1000 with 2200 pages back and
// 4000 given in 9.5.
template <int N>
__global__ __launch_bounds__(N) void k_pages_plan(PagesDev c, const int* fresh, int tokens, int* starts, int* slots,
                                                  int* positions, int place) {
  __shared__ int lds[4][N / 64], at[N], held[N], begin[N + 1];
  const int tid = threadIdx.x, P = 1 << c.lp, limit = c.max_pages << c.lp;
  // of the first N sequences
  const int fresh0 = tid < c.seqs ? fresh[tid] : 0;
  int rows0 = tid < c.seqs ? pg_rows(c, tid) : 0;
  int count = min(max(c.free[0], 0), c.pages);
  // what has ended gives its pages back, in order
  for (int s0 = 0; s0 < c.seqs; s0 += N) {
    const int s = s0 + tid, n = min(N, c.seqs - s0);
    const bool ends = s < c.seqs && (s0 ? fresh[s] : fresh0) < 0;
    if (!__syncthreads_or(ends)) continue;
    const int back = ends ? ((s0 ? pg_rows(c, s) : rows0) + P - 1) >> c.lp : 0;
    const int2 sum = plan_scan<N>(min(back, c.pages + 1), c.pages + 1, lds[0]);
    at[tid] = sum.x;
    if (ends) {
      int* st = c.state + (size_t)s * PG_STATE;
      st[PG_ROWS] = st[PG_REFUSED] = st[PG_FROM] = 0;
      if (s0 == 0) rows0 = 0;
    }
    __syncthreads();
    const int all = min(sum.y, c.pages - count);
    for (int i = tid; i < all; i += kRuns * N) {
      int x[kRuns], j[kRuns], page[kRuns];
#pragma unroll
      for (int r = 0; r < kRuns; r++) x[r] = min(i + r * N, all - 1);
      last_from<kRuns>(at, n, x, j);
#pragma unroll
      for (int r = 0; r < kRuns; r++)
        page[r] = c.table[(size_t)(s0 + j[r]) * c.max_pages + min(x[r] - at[j[r]], c.max_pages - 1)];
#pragma unroll
      for (int r = 0; r < kRuns; r++)
        if (i + r * N < all) c.free[1 + count + x[r]] = page[r];
    }
    count += all;
    __syncthreads();
  }
  // the others in order, as long as there are pages
  int first = 0, taken = 0, given = 0;  // of the sequences before: rows, pages that they lacked, pages that they got
  for (int s0 = 0; s0 < c.seqs; s0 += N) {
    const int s = s0 + tid, n = min(N, c.seqs - s0);
    const int want = s < c.seqs ? max(s0 ? fresh[s] : fresh0, 0) : 0;
    const int rows = s0 ? (s < c.seqs ? pg_rows(c, s) : 0) : rows0;
    const int2 sum = plan_scan<N>(min(want, tokens + 1), tokens + 1, lds[1]);
    const int start = min(first + sum.x, tokens + 1), end = min(start + min(want, tokens + 1), tokens + 1);
    const bool room = want == 0 || (end <= tokens && want <= limit - rows);
    const int has = (rows + P - 1) >> c.lp, need = room ? ((rows + want + P - 1) >> c.lp) - has : 0;
    const int2 pg = plan_scan<N>(min(need, c.pages + 1), c.pages + 1, lds[2]);
    const int before = min(taken + pg.x, c.pages + 1);
    const bool ok = room && (need == 0 || before + need <= count);
    at[tid] = before;
    held[tid] = has;
    begin[tid] = min(start, tokens);
    first = min(first + sum.y, tokens + 1);
    if (tid == 0) begin[n] = min(first, tokens);
    if (s < c.seqs) {
      int* st = c.state + (size_t)s * PG_STATE;
      st[PG_FROM] = ok ? rows : -1;
      if (ok) st[PG_ROWS] = rows + want;
      else st[PG_REFUSED] = st[PG_REFUSED] > 0x7fffffff - want ? 0x7fffffff : st[PG_REFUSED] + want;
      starts[s] = min(start, tokens);
    }
    // those that get pages come before those that do not: what is given is a run of the stack
    int most = taken + pg.y;
    if (most > count) {
      most = ok && need ? before + need : given;
#pragma unroll
      for (int d = 32; d; d /= 2) most = max(most, __shfl_xor(most, d));
      if ((tid & 63) == 0) lds[3][tid >> 6] = most;
      __syncthreads();
      most = given;
#pragma unroll
      for (int i = 0; i < N / 64; i++) most = max(most, lds[3][i]);
    }
    __syncthreads();
    for (int i = given + tid; i < most; i += kRuns * N) {
      int x[kRuns], j[kRuns], page[kRuns];
#pragma unroll
      for (int r = 0; r < kRuns; r++) {
        x[r] = min(i + r * N, most - 1);
        page[r] = c.free[count - x[r]];
      }
      last_from<kRuns>(at, n, x, j);
#pragma unroll
      for (int r = 0; r < kRuns; r++)
        if (i + r * N < most)
          c.table[(size_t)(s0 + j[r]) * c.max_pages + min(held[j[r]] + x[r] - at[j[r]], c.max_pages - 1)] = page[r];
    }
    taken = min(taken + pg.y, c.pages + 1);
    given = most;
    __syncthreads();
    if (place) {  // one round
      for (int i = tid; i < tokens; i += N) {
        int x = n;
        if (i < begin[n]) {
          last_from<1>(begin, n, &i, &x);
          plan_row(c, x, begin[x], i, slots, positions);
        } else {
          slots[i] = -1;
          if (positions) positions[i] = -1;
        }
      }
    }
  }
  if (tid == 0) {
    starts[c.seqs] = min(first, tokens);
    c.free[0] = count - given;
  }
}

constexpr int kSlotRows = 256, kSlotSeqs = 1024;

// The rows' slots, 256 rows to a workgroup: 64 candidates at a time say which sequences have the first and the last of them,
// and the starts of those go to LDS for each row's search. (A search of every row in memory: 4.9 us where this takes 4.0.)
__global__ __launch_bounds__(kSlotRows) void k_pages_slots(PagesDev c, const int* starts, int tokens, int* slots,
                                                           int* positions) {
  __shared__ int begin[kSlotSeqs];
  const int i0 = blockIdx.x * kSlotRows, i = i0 + threadIdx.x, lane = threadIdx.x & 63, all = starts[c.seqs];
  // 64 candidates at a time, for the first row and the last side by side
  int lo[2] = {0, 0};
  for (int range = c.seqs; range > 1;) {
    const int step = (range + 63) / 64;
#pragma unroll
    for (int z = 0; z < 2; z++) {
      const int row = z ? min(i0 + kSlotRows, tokens) - 1 : i0, x = lo[z] + lane * step;
      const bool in = lane * step < range && x < c.seqs && gmem(starts)[min(x, c.seqs - 1)] <= row;
      const unsigned long long m = __ballot(in);
      lo[z] += m ? (63 - __builtin_clzll(m)) * step : 0;
    }
    range = step;
  }
  const int s0 = lo[0], n = lo[1] - lo[0] + 1;
  const bool fits = n > 0 && n <= kSlotSeqs;
  if (fits)
    for (int x = threadIdx.x; x < n; x += kSlotRows) begin[x] = starts[s0 + x];
  __syncthreads();
  if (i >= tokens) return;
  if (i >= all) {
    slots[i] = -1;
    if (positions) positions[i] = -1;
    return;
  }
  int x;
  if (fits) {
    last_from<1>(begin, n, &i, &x);
    plan_row(c, s0 + x, begin[x], i, slots, positions);
  } else {  // more sequences, most of them without rows
    last_from<1>(starts, c.seqs, &i, &x);
    plan_row(c, x, starts[x], i, slots, positions);
  }
}

// Eight elements of a row in the cache's type, as bits. vec: the rows' strides and pointer allow 16-byte loads, which are
// made with the non-temporal hint: rows are read once (194 MB 50.8 us a pass without, 47.3 with).
__device__ __forceinline__ uint4 row_bits(const KvRows& r, long long at, bool vec) {
  uint32_t w[4];
  if (r.f16) {
    const uint16_t* p = (const uint16_t*)r.p + at;
    if (vec) return gload_u4_nt(p);
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)gmem(p)[2 * i] | (uint32_t)gmem(p)[2 * i + 1] << 16;
  } else {
    const float* p = (const float*)r.p + at;
    float x[8];
    if (vec) {
      const uint4 a = gload_u4_nt(p), b = gload_u4_nt(p + 4);
      x[0] = __uint_as_float(a.x), x[1] = __uint_as_float(a.y), x[2] = __uint_as_float(a.z), x[3] = __uint_as_float(a.w);
      x[4] = __uint_as_float(b.x), x[5] = __uint_as_float(b.y), x[6] = __uint_as_float(b.z), x[7] = __uint_as_float(b.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = gmem(p)[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Whether any of eight 16-bit values is not finite: has all bits of the exponent.
template <int BF16>
__device__ __forceinline__ bool not_finite(uint4 x) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) bad |= (w[i] & kExp) == kExp || (w[i] >> 16 & kExp) == kExp;
  return bad;
}

constexpr int kHalo = 3;  // rows of the next workgroup that a run of four may take in

// How a row of V leaves: not at all (no slot, or with another row's), alone, with the three behind it, or with those and the
// four that are 8 on.
enum { kNot, kAlone, kFour, kEight };

// A workgroup per kTile rows of the batch and KV head. The rows come in whole lines and go to LDS, from where K leaves 16
// bytes at a time and V, the four positions of an element that lie side by side, 8 bytes, or 16 with the four that are 8
// on. Such a run belongs to its first row's workgroup; what is in no run, such as single rows of many sequences, goes 2 bytes
// at a time. A row of K or V that is not finite becomes a K of NaN and a V of zeros: whoever sees it gets NaN, and whoever
// does not, nothing of it. Bound by its instructions more than by memory: 24000 rows of 8 KV heads of 128, 194 MB, in
// about 42 us; with every element's way looked at by itself 48, an element instead of two to a thread 66, a wave to a row 81.
template <int D, int BF16, int kTile>
__global__ __launch_bounds__(256) void k_pages_append(PagesDev c, KvRows k, KvRows v, const int* slots, int tokens,
                                                      int vec) {
  constexpr int C = D / 8, kPitch = D + 8;  // chunks of a row, and a row in LDS
  __shared__ __align__(16) uint16_t ks[kTile][kPitch], vs[kTile + kHalo][kPitch];
  __shared__ int at[kTile + 2 * kHalo], bad[kTile + kHalo], how[kTile], block[kTile], k_at[kTile];
  const int tid = threadIdx.x, h = blockIdx.x % c.kvh, i0 = blockIdx.x / c.kvh * kTile;
  if (tid < kTile + 2 * kHalo) {  // slots from row i0 - kHalo on, -1 where there is none
    const int i = i0 - kHalo + tid, slot = i >= 0 && i < tokens ? slots[i] : -1;
    at[tid] = (unsigned)slot < (unsigned)c.pages << c.lp ? slot : -1;
  }
  if (tid < kTile + kHalo) bad[tid] = 0;
  __syncthreads();
  bool any = false;
#pragma unroll 2
  for (int x = tid; x < (kTile + kHalo) * C; x += 256) {
    const int j = x / C, e = x % C * 8, i = i0 + j;
    if (at[j + kHalo] < 0) continue;
    const uint4 a = row_bits(k, i * k.pos + h * k.head + e, vec & 1), b = row_bits(v, i * v.pos + h * v.head + e, vec & 2);
    if (j < kTile) *reinterpret_cast<uint4*>(&ks[j][e]) = a;
    *reinterpret_cast<uint4*>(&vs[j][e]) = b;
    if (not_finite<BF16>(a) || not_finite<BF16>(b)) bad[j] = 1, any = true;
  }
  if (tid < kTile) {
    const int* s = at + kHalo;
    const int j = tid, slot = s[j], t = slot % kPgBlock;
    auto run = [&](int i) {  // of four positions from a multiple of four on
      return s[i] >= 0 && s[i] % 4 == 0 && s[i + 1] == s[i] + 1 && s[i + 2] == s[i] + 2 && s[i + 3] == s[i] + 3;
    };
    int way = slot < 0 ? kNot : kAlone;
    if (slot >= 0 && run(j)) {
      way = kFour;
      if (t % 16 < 8 && j + 8 < kTile && s[j + 8] == slot + 8 && run(j + 8)) way = kEight;
      if (t % 16 >= 8 && j >= 8 && s[j - 8] == slot - 8 && run(j - 8)) way = kNot;
    } else if (slot >= 0) {
#pragma unroll
      for (int z = 1; z <= kHalo; z++)
        if (t % 4 == z && s[j - z] == slot - z && run(j - z)) way = kNot;
    }
    how[j] = way;
    const int pos = slot & ((1 << c.lp) - 1);
    block[j] = slot < 0 ? -1 : pg_block(c, slot >> c.lp, h, pos / kPgBlock);
    k_at[j] = t;
  }
  if (__syncthreads_or(any)) {
    for (int x = tid; x < (kTile + kHalo) * C; x += 256) {
      const int j = x / C, e = x % C * 8;
      if (!bad[j]) continue;
      if (j < kTile) *reinterpret_cast<uint4*>(&ks[j][e]) = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      *reinterpret_cast<uint4*>(&vs[j][e]) = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }
  for (int x = tid; x < kTile * C; x += 256) {
    const int j = x % kTile, e = x / kTile * 8, b = block[j];
    if (b >= 0)
      *reinterpret_cast<uint4*>(c.k + (size_t)b * (kPgBlock * D) + pg_k_place(k_at[j], e)) =
          *reinterpret_cast<const uint4*>(&ks[j][e]);
  }
  for (int x = tid; x < kTile * (D / 2); x += 256) {
    const int j = x / (D / 2), e = x % (D / 2) * 2, way = how[j];
    if (way == kNot) continue;
    uint16_t* to = c.v + (size_t)block[j] * (kPgBlock * D) + pg_v_place(D, k_at[j], e);
    auto pair = [&](int i) { return *reinterpret_cast<const uint32_t*>(&vs[i][e]); };
    if (way == kAlone) {
      const uint32_t w = pair(j);
      to[0] = (uint16_t)w;
      to[8] = (uint16_t)(w >> 16);
      continue;
    }
    auto quad = [&](int i, uint2* a, uint2* b) {  // four rows' elements e and e + 1
      const uint32_t w[4] = {pair(i), pair(i + 1), pair(i + 2), pair(i + 3)};
      *a = make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x05040100u), __builtin_amdgcn_perm(w[3], w[2], 0x05040100u));
      *b = make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x07060302u), __builtin_amdgcn_perm(w[3], w[2], 0x07060302u));
    };
    uint2 a, b;
    quad(j, &a, &b);
    if (way == kEight) {
      uint2 p, q;
      quad(j + 8, &p, &q);
      *reinterpret_cast<uint4*>(to) = make_uint4(a.x, a.y, p.x, p.y);
      *reinterpret_cast<uint4*>(to + 8) = make_uint4(b.x, b.y, q.x, q.y);
    } else {
      *reinterpret_cast<uint2*>(to) = a;
      *reinterpret_cast<uint2*>(to + 8) = b;
    }
  }
}

}  // namespace

hipError_t launch_pages_clear(hipStream_t s, const PagesDev& c) {
  const int n = c.seqs * PG_STATE > c.pages ? c.seqs * PG_STATE : c.pages;
  klaunch(k_pages_clear, (n + 255) / 256, 256, 0, s, c);
  return hipGetLastError();
}

hipError_t launch_pages_plan(hipStream_t s, const PagesDev& c, const int* fresh, int tokens, int* starts, int* slots,
                             int* positions) {
  // Small plans with fewer threads, whose barriers cost less; up to four rows to a thread without a second launch.
  const int small = c.seqs <= 256 && tokens <= 1024, place = small || (c.seqs <= 1024 && tokens <= 4096);
  if (small) klaunch(k_pages_plan<256>, 1, 256, 0, s, c, fresh, tokens, starts, slots, positions, place);
  else klaunch(k_pages_plan<1024>, 1, 1024, 0, s, c, fresh, tokens, starts, slots, positions, place);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!place && tokens)
    klaunch(k_pages_slots, (tokens + kSlotRows - 1) / kSlotRows, kSlotRows, 0, s, c, starts, tokens, slots, positions);
  return hipGetLastError();
}

hipError_t launch_pages_append(hipStream_t s, const PagesDev& c, KvRows k, KvRows v, const int* slots, int tokens) {
  const int vec = wide_rows(k) | wide_rows(v) << 1;
  // 8 rows to a workgroup where 32 would leave compute units without any
  const int tile = (tokens + 31) / 32 * (long long)c.kvh < 256 ? 8 : 32;
  const unsigned grid = (unsigned)((tokens + tile - 1) / tile) * c.kvh;  // at most 2^22 + 255
#define APPEND(DD, BB, TT)                   \
  if (c.d == DD && c.bf16 == BB && tile == TT) \
    klaunch(k_pages_append<DD, BB, TT>, grid, 256, 0, s, c, k, v, slots, tokens, vec);
  APPEND(64, 0, 8) APPEND(64, 1, 8) APPEND(128, 0, 8) APPEND(128, 1, 8)
  APPEND(64, 0, 32) APPEND(64, 1, 32) APPEND(128, 0, 32) APPEND(128, 1, 32)
#undef APPEND
  return hipGetLastError();
}

}  // namespace moert

// ---- C entry points --------------------------------------------------------------------------------------------
using namespace moert;

namespace {

constexpr int kPgMaxLen = 1 << 20, kPgMaxSeqs = 65535, kPgMaxHeads = 256, kPgMaxTokens = 1 << 24;

enum { PG_POOL = 1, PG_TABLE = 2, PG_FREE = 4 };  // buffers that a call uses, beside the state

int view(const char* what, const moert_pages* c, int uses, PagesDev* d) {
  KV_CFG(c, "%s: null cache", what);
  KV_CFG(c->seqs >= 1 && c->seqs <= kPgMaxSeqs && c->kv_heads >= 1 && c->kv_heads <= kPgMaxHeads &&
             (long long)c->seqs * c->kv_heads <= 1 << 20 && (c->head_dim == 64 || c->head_dim == 128),
         "%s: %d sequences, %d KV heads of %d", what, c->seqs, c->kv_heads, c->head_dim);
  KV_CFG(c->page >= kPgBlock && c->page <= 256 && (c->page & (c->page - 1)) == 0, "%s: pages of %d positions", what,
         c->page);
  KV_CFG(c->pages >= 1 && c->max_pages >= 1 && (long long)c->pages * c->page <= 1 << 30 &&
             (long long)c->pages * c->page * c->kv_heads <= 1ll << 35 &&
             (long long)c->max_pages * c->page <= kPgMaxLen && (long long)c->seqs * c->max_pages <= 1 << 30,
         "%s: %d pages of %d positions, %d of a sequence", what, c->pages, c->page, c->max_pages);
  KV_CFG(c->dtype == MOERT_F16 || c->dtype == MOERT_BF16, "%s: a cache of dtype %d", what, c->dtype);
  KV_CFG(c->state_dev && (!(uses & PG_POOL) || (c->k_dev && c->v_dev)) && (!(uses & PG_TABLE) || c->table_dev) &&
             (!(uses & PG_FREE) || c->free_dev),
         "%s: a null buffer", what);
  const uintptr_t wide = (uintptr_t)c->k_dev | (uintptr_t)c->v_dev;
  const uintptr_t words = (uintptr_t)c->table_dev | (uintptr_t)c->state_dev | (uintptr_t)c->free_dev;
  KV_CFG(wide % 16 == 0 && words % 4 == 0, "%s: K and V are aligned to 16 bytes, the others to 4", what);
  int lp = 5;
  while (1 << lp < c->page) lp++;
  *d = PagesDev{c->seqs,  c->kv_heads, c->head_dim,  c->pages,     c->max_pages, lp, c->dtype == MOERT_BF16,
                c->k_dev, c->v_dev,    c->table_dev, c->state_dev, c->free_dev};
  return MOERT_OK;
}

// Types of rows that go with the cache's.
int types_of(const PagesDev& d) { return d.bf16 ? 1 << MOERT_BF16 : 1 << MOERT_F32 | 1 << MOERT_F16; }

int tokens_ok(const char* what, int tokens) {
  KV_CFG(tokens >= 0 && tokens <= kPgMaxTokens, "%s: %d rows", what, tokens);
  return MOERT_OK;
}

int heads_ok(const char* what, const PagesDev& d, int heads, int tokens) {
  KV_CFG(heads >= 1 && heads % d.kvh == 0 && heads / d.kvh <= 64, "%s: %d query heads over %d KV heads", what, heads,
         d.kvh);
  KV_CFG((long long)d.seqs * heads <= 1 << 24, "%s: %d sequences x %d heads", what, d.seqs, heads);
  KV_TRY(tokens_ok(what, tokens));
  KV_CFG((long long)tokens * heads <= 1 << 27, "%s: %d rows x %d heads", what, tokens, heads);
  return MOERT_OK;
}

int workspace_ok(const char* what, size_t need, const void* ws, size_t bytes) {
  KV_CFG(bytes >= need && (!need || (ws && (uintptr_t)ws % 16 == 0)),
         "%s: a workspace of %zu bytes aligned to 16 is needed, got %zu", what, need, bytes);
  return MOERT_OK;
}

int ints_ok(const char* what, const int* p) {
  KV_CFG(p && (uintptr_t)p % 4 == 0, "%s: a null or unaligned array", what);
  return MOERT_OK;
}

// What an attention is called with.
int queries(const char* what, const PagesDev& d, int heads, float scale, const moert_rows* q, const moert_rows* out,
            int tokens, KvRows* qr, KvRows* orow) {
  KV_TRY(heads_ok(what, d, heads, tokens));
  KV_CFG(scale - scale == 0.0f, "%s: scale %g", what, (double)scale);
  KV_TRY(rows(what, q, types_of(d), 1, tokens, heads, d.d, false, qr));
  KV_TRY(rows(what, out, types_of(d), 1, tokens, heads, d.d, true, orow));
  KV_CFG(q->dtype == out->dtype, "%s: q of dtype %d, out of %d", what, q->dtype, out->dtype);
  return MOERT_OK;
}

}  // namespace

extern "C" {

int moert_pages_clear(const moert_pages* c, void* stream) {
  PagesDev d;
  KV_TRY(view("pages_clear", c, PG_FREE, &d));
  OnDevice on;
  KV_TRY(on.enter("pages_clear", d.state));
  KV_HIP(launch_pages_clear((hipStream_t)stream, d));
  return MOERT_OK;
}

int moert_pages_plan(const moert_pages* c, const int* new_dev, int tokens, int* starts_dev, int* slots_dev,
                     int* positions_dev, void* stream) {
  PagesDev d;
  KV_TRY(view("pages_plan", c, PG_TABLE | PG_FREE, &d));
  KV_TRY(tokens_ok("pages_plan", tokens));
  KV_TRY(ints_ok("pages_plan", new_dev));
  KV_TRY(ints_ok("pages_plan", starts_dev));
  if (tokens) KV_TRY(ints_ok("pages_plan", slots_dev));
  KV_CFG((uintptr_t)positions_dev % 4 == 0, "pages_plan: a null or unaligned array");
  OnDevice on;
  KV_TRY(on.enter("pages_plan", d.state));
  KV_HIP(launch_pages_plan((hipStream_t)stream, d, new_dev, tokens, starts_dev, slots_dev, positions_dev));
  return MOERT_OK;
}

int moert_pages_append(const moert_pages* c, const moert_rows* k, const moert_rows* v, const int* slots_dev,
                       int tokens, void* stream) {
  PagesDev d;
  KvRows kr, vr;
  KV_TRY(view("pages_append", c, PG_POOL, &d));
  KV_TRY(tokens_ok("pages_append", tokens));
  KV_CFG((long long)tokens * d.kvh <= 1 << 27, "pages_append: %d rows x %d KV heads", tokens, d.kvh);
  if (!tokens) return MOERT_OK;
  KV_TRY(ints_ok("pages_append", slots_dev));
  KV_TRY(rows("pages_append", k, types_of(d), 1, tokens, d.kvh, d.d, false, &kr));
  KV_TRY(rows("pages_append", v, types_of(d), 1, tokens, d.kvh, d.d, false, &vr));
  KV_CFG(k->dtype == v->dtype, "pages_append: K of dtype %d, V of %d", k->dtype, v->dtype);
  OnDevice on;
  KV_TRY(on.enter("pages_append", d.k));
  KV_HIP(launch_pages_append((hipStream_t)stream, d, kr, vr, slots_dev, tokens));
  return MOERT_OK;
}

int moert_pages_workspace(const moert_pages* c, int heads, int tokens, size_t* bytes) {
  PagesDev d;
  KV_TRY(view("pages_workspace", c, 0, &d));
  KV_CFG(bytes, "pages_workspace: null bytes");
  KV_TRY(heads_ok("pages_workspace", d, heads, tokens));
  *bytes = pages_workspace(d, heads, tokens);
  return MOERT_OK;
}

int moert_pages_attend(const moert_pages* c, int heads, float scale, const moert_rows* q, const moert_rows* out,
                       const int* starts_dev, int tokens, void* ws_dev, size_t ws_bytes, void* stream) {
  PagesDev d;
  KvRows qr, orow;
  KV_TRY(view("pages_attend", c, PG_POOL | PG_TABLE, &d));
  KV_TRY(queries("pages_attend", d, heads, scale, q, out, tokens, &qr, &orow));
  if (starts_dev) KV_TRY(ints_ok("pages_attend", starts_dev));
  else KV_CFG(tokens == d.seqs, "pages_attend: %d rows of %d sequences, without starts", tokens, d.seqs);
  KV_TRY(workspace_ok("pages_attend", pages_workspace(d, heads, 0), ws_dev, ws_bytes));
  if (!tokens) return MOERT_OK;
  OnDevice on;
  KV_TRY(on.enter("pages_attend", d.k));
  KV_HIP(launch_pages_attend((hipStream_t)stream, d, heads, scale, qr, orow, starts_dev, tokens, ws_dev, ws_bytes));
  return MOERT_OK;
}

int moert_pages_prompt(const moert_pages* c, int heads, float scale, const moert_rows* q, const moert_rows* out,
                       const int* starts_dev, int tokens, int least, void* ws_dev, size_t ws_bytes, void* stream) {
  PagesDev d;
  KvRows qr, orow;
  KV_TRY(view("pages_prompt", c, PG_POOL | PG_TABLE, &d));
  KV_TRY(queries("pages_prompt", d, heads, scale, q, out, tokens, &qr, &orow));
  KV_TRY(ints_ok("pages_prompt", starts_dev));
  KV_CFG(least >= 1, "pages_prompt: sequences of at least %d rows", least);
  KV_TRY(workspace_ok("pages_prompt", pages_workspace(d, heads, tokens), ws_dev, ws_bytes));
  if (!tokens) return MOERT_OK;
  OnDevice on;
  KV_TRY(on.enter("pages_prompt", d.k));
  KV_HIP(launch_pages_prompt((hipStream_t)stream, d, heads, scale, qr, orow, starts_dev, tokens, least, ws_dev,
                              ws_bytes));
  return MOERT_OK;
}

int moert_pages_lengths(const moert_pages* c, int seq0, int n_seqs, int* lengths, void* stream) {
  PagesDev d;
  KV_TRY(view("pages_lengths", c, 0, &d));
  KV_CFG(seq0 >= 0 && n_seqs >= 1 && n_seqs <= d.seqs - seq0, "pages_lengths: sequences %d + %d of %d", seq0, n_seqs,
         d.seqs);
  KV_CFG(lengths, "pages_lengths: null lengths");
  OnDevice on;
  KV_TRY(on.enter("pages_lengths", d.state));
  hipStream_t s = (hipStream_t)stream;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  KV_HIP(hipStreamIsCapturing(s, &cs));
  KV_CFG(cs == hipStreamCaptureStatusNone, "pages_lengths: the stream is being captured");
  int refused = 0, part[64 * PG_STATE];
  for (int i = 0; i < n_seqs; i += 64) {
    const int m = n_seqs - i < 64 ? n_seqs - i : 64;
    KV_HIP(hipMemcpyAsync(part, d.state + (size_t)(seq0 + i) * PG_STATE, (size_t)m * PG_STATE * 4,
                          hipMemcpyDeviceToHost, s));
    KV_HIP(hipStreamSynchronize(s));
    for (int j = 0; j < m; j++) {
      lengths[i + j] = part[j * PG_STATE + PG_ROWS];
      if (part[j * PG_STATE + PG_REFUSED] && !refused) refused = 1 + i + j;
    }
  }
  if (refused)
    return set_error(MOERT_E_FULL, "pages_lengths: sequence %d has been refused rows for want of room",
                     seq0 + refused - 1);
  return MOERT_OK;
}

}  // extern "C"
