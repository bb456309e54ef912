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

constexpr int kPlan = 1024;  // threads of a plan, and sequences that it looks at together

// Sums over the threads before this one and over all of them, none above `most` (of terms in [0, most], most < 2^30).
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
  for (int i = 0; i < kPlan / 64; i++) {
    if (i == w) before = all;
    all = min(all + lds[i], most);
  }
  __syncthreads();
  const int up = __shfl_up(sum, 1);
  return make_int2(min(before + (lane ? up : 0), most), all);
}

// The last i in [0, n) with at[i] <= x (at[0] <= x, at not falling).
__device__ __forceinline__ int last_from(const int* at, int n, int x) {
  int lo = 0;
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Slot and position of row i of the batch. at: where the rows of sequences s0 .. s0 + n - 1 start, and end.
__device__ __forceinline__ void plan_row(const PagesDev& c, const int* at, int n, int s0, int i, int* slots,
                                         int* positions) {
  int slot = -1, pos = -1;
  if (i < at[n]) {
    const int x = last_from(at, n, i), s = s0 + x, from = c.state[(size_t)s * PG_STATE + PG_FROM];
    if (from >= 0) {
      pos = from + i - at[x];
      const int page = c.table[(size_t)s * c.max_pages + (pos >> c.lp)];
      if ((unsigned)page < (unsigned)c.pages) slot = (page << c.lp) + (pos & ((1 << c.lp) - 1));
    }
  }
  slots[i] = slot;
  if (positions) positions[i] = pos;
}

// One workgroup takes the sequences 1024 at a time: sums over them, in order, say where the pages of each lie on the free
// stack, and all threads together move the pages. With `place` also the rows' slots.
__global__ __launch_bounds__(kPlan) void k_pages_plan(PagesDev c, const int* fresh, int tokens, int* starts, int* slots,
                                                      int* positions, int place) {
  __shared__ int lds[kPlan / 64], at[kPlan + 1], held[kPlan];
  const int tid = threadIdx.x, P = 1 << c.lp, limit = c.max_pages << c.lp;
  int count = min(max(c.free[0], 0), c.pages);
  // what has ended gives its pages back, in order
  for (int s0 = 0; s0 < c.seqs; s0 += kPlan) {
    const int s = s0 + tid, n = min(kPlan, c.seqs - s0);
    const bool ends = s < c.seqs && fresh[s] < 0;
    if (!__syncthreads_or(ends)) continue;
    const int back = ends ? (pg_rows(c, s) + P - 1) >> c.lp : 0;
    const int2 sum = plan_scan(min(back, c.pages + 1), c.pages + 1, lds);
    at[tid] = sum.x;
    if (ends) {
      int* st = c.state + (size_t)s * PG_STATE;
      st[PG_ROWS] = st[PG_REFUSED] = st[PG_FROM] = 0;
    }
    __syncthreads();
    const int all = min(sum.y, c.pages - count);
    for (int i = tid; i < all; i += kPlan) {
      const int x = last_from(at, n, i);
      c.free[1 + count + i] = c.table[(size_t)(s0 + x) * c.max_pages + min(i - at[x], c.max_pages - 1)];
    }
    count += all;
    __syncthreads();
  }
  // the others in order, as long as there are pages
  int first = 0, taken = 0, given = 0;  // of the sequences before: rows, pages that they lacked, pages that they got
  for (int s0 = 0; s0 < c.seqs; s0 += kPlan) {
    const int s = s0 + tid, n = min(kPlan, c.seqs - s0);
    const int want = s < c.seqs ? max(fresh[s], 0) : 0, rows = s < c.seqs ? pg_rows(c, s) : 0;
    const int2 sum = plan_scan(min(want, tokens + 1), tokens + 1, lds);
    const int start = min(first + sum.x, tokens + 1), end = min(start + min(want, tokens + 1), tokens + 1);
    const bool room = want == 0 || (end <= tokens && want <= limit - rows);
    const int has = (rows + P - 1) >> c.lp, need = room ? ((rows + want + P - 1) >> c.lp) - has : 0;
    const int2 pg = plan_scan(min(need, c.pages + 1), c.pages + 1, lds);
    const int before = min(taken + pg.x, c.pages + 1);
    const bool ok = room && (need == 0 || before + need <= count);
    at[tid] = before;
    held[tid] = has;
    if (s < c.seqs) {
      int* st = c.state + (size_t)s * PG_STATE;
      st[PG_FROM] = ok ? rows : -1;
      if (ok) st[PG_ROWS] = rows + want;
      else st[PG_REFUSED] = st[PG_REFUSED] > 0x7fffffff - want ? 0x7fffffff : st[PG_REFUSED] + want;
      starts[s] = min(start, tokens);
    }
    // those that get pages come before those that do not: what is given is a run of the stack
    const int mine = ok && need ? before + need : 0;
    __syncthreads();
    int most = mine;
#pragma unroll
    for (int d = 32; d; d /= 2) most = max(most, __shfl_xor(most, d));
    if ((tid & 63) == 0) lds[tid >> 6] = most;
    __syncthreads();
    most = given;
#pragma unroll
    for (int i = 0; i < kPlan / 64; i++) most = max(most, lds[i]);
    for (int i = given + tid; i < most; i += kPlan) {
      const int x = last_from(at, n, i);
      c.table[(size_t)(s0 + x) * c.max_pages + min(held[x] + i - at[x], c.max_pages - 1)] = c.free[count - i];
    }
    first = min(first + sum.y, tokens + 1);
    taken = min(taken + pg.y, c.pages + 1);
    given = most;
    __syncthreads();
    if (place) {  // one round
      if (tid == 0) at[n] = min(first, tokens);
      if (tid < n) at[tid] = min(start, tokens);
      __syncthreads();
      for (int i = tid; i < tokens; i += kPlan) plan_row(c, at, n, s0, i, slots, positions);
    }
  }
  if (tid == 0) {
    starts[c.seqs] = min(first, tokens);
    c.free[0] = count - given;
  }
}

__global__ __launch_bounds__(256) void k_pages_slots(PagesDev c, const int* starts, int tokens, int* slots,
                                                     int* positions) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < tokens) plan_row(c, starts, c.seqs, 0, i, slots, positions);
}

// An element in the cache's type, as bits.
template <int BF16>
__device__ __forceinline__ uint16_t held_bits(const KvRows& r, long long at) {
  if (BF16) return ((const uint16_t*)r.p)[at];
  return r.f16 ? ((const uint16_t*)r.p)[at] : f2h(((const float*)r.p)[at]);
}

// A wave per row and KV head. A row of K or V that is not finite becomes a K of NaN and a V of zeros: whoever sees it
// gets NaN, and whoever does not, nothing of it.
template <int BF16>
__global__ __launch_bounds__(256) void k_pages_append(PagesDev c, KvRows k, KvRows v, const int* slots, int tokens) {
  const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= (long long)tokens * c.kvh) return;
  const int lane = threadIdx.x & 63, i = (int)(u / c.kvh), h = (int)(u % c.kvh), slot = slots[i];
  if ((unsigned)slot >= (unsigned)c.pages << c.lp) return;
  const int page = slot >> c.lp, pos = slot & ((1 << c.lp) - 1), t = pos % kPgBlock;
  const size_t at = (size_t)pg_block(c, page, h, pos / kPgBlock) * (kPgBlock * c.d);
  constexpr int kInf = BF16 ? 0x7f80 : 0x7c00;
  bool bad = false;
  uint16_t x[2], y[2];
  for (int j = 0; j < c.d / 64; j++) {
    x[j] = held_bits<BF16>(k, i * k.pos + h * k.head + lane + 64 * j);
    y[j] = held_bits<BF16>(v, i * v.pos + h * v.head + lane + 64 * j);
    bad |= (x[j] & 0x7fff) >= kInf || (y[j] & 0x7fff) >= kInf;
  }
  bad = __any(bad);
  for (int j = 0; j < c.d / 64; j++) {
    c.k[at + pg_k_place(t, lane + 64 * j)] = bad ? 0x7fff : x[j];
    c.v[at + pg_v_place(c.d, t, lane + 64 * j)] = bad ? 0 : y[j];
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
  const int place = c.seqs <= kPlan && tokens <= 4096;
  klaunch(k_pages_plan, 1, kPlan, 0, s, c, fresh, tokens, starts, slots, positions, place);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!place && tokens) klaunch(k_pages_slots, (tokens + 255) / 256, 256, 0, s, c, starts, tokens, slots, positions);
  return hipGetLastError();
}

hipError_t launch_pages_append(hipStream_t s, const PagesDev& c, KvRows k, KvRows v, const int* slots, int tokens) {
  const unsigned grid = (unsigned)(((long long)tokens * c.kvh + 3) / 4);
  if (c.bf16) klaunch(k_pages_append<1>, grid, 256, 0, s, c, k, v, slots, tokens);
  else klaunch(k_pages_append<0>, grid, 256, 0, s, c, k, v, slots, tokens);
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
