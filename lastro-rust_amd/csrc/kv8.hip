// The 8-bit K/V cache: append, read back, eviction, and the C entry points (kv8_attn.hip has the attention).
#include "kv8.h"

#include "../../include/moert.h"
#include "launch.h"

namespace moert {

int set_error(int code, const char* fmt, ...);

namespace {

// Rows t < 32 of one block, K or V, as fp16 in LDS: two elements apart from row to row more than the row has, so that
// a column's elements lie in different banks.
template <int D>
struct BlockLds {
  uint16_t x[kKvBlock][D + 2];
};

__device__ __forceinline__ uint16_t row_elem(const KvRows& r, long long at) {
  return r.f16 ? gmem((const uint16_t*)r.p)[at] : f2h(gmem((const float*)r.p)[at]);
}

// round(x / s), ties to even, of the exact quotient. x * inv is off by less than one step near a tie; the residual
// x - q s (one fma) decides: next to a tie it is a multiple of ulp(s) / 2 below s, so it is exact there.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float q = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
  if (r > h || (r == h && ((int)q & 1))) q += 1.0f;
  else if (r < -h || (r == -h && ((int)q & 1))) q -= 1.0f;
  return (int)q;
}

// Codes the 32 rows in `b` (one wave, K or V) into `codes` and returns the scale.
template <int D, bool V>
__device__ float code_block(const BlockLds<D>& b, int lane, uint8_t* codes) {
  int top = 0;
  for (int i = lane; i < kKvBlock * D; i += 64) top = max(top, b.x[i / D][i % D] & 0x7fff);
#pragma unroll
  for (int m = 32; m; m >>= 1) top = max(top, __shfl_xor(top, m));
  const float a = h2f((uint16_t)top);
  const bool bad = top >= 0x7c00;
  const float s = bad ? __int_as_float(0x7fc00000) : top ? a / 127.0f : 1.0f, inv = 1.0f / s;
  for (int i = lane; i < kKvBlock * D / 8; i += 64) {  // 8 codes, one store
    uint32_t w[2] = {0x80808080u, 0x80808080u};
    if (!bad) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        // V: i = (r * 4 + g) * U + u, element r U + u, positions 4 g + j and 16 + 4 g + j
        constexpr int U = D / 16;
        const int t = V ? i / U % 4 * 4 + (j & 3) + 16 * (j >> 2) : i * 8 / D;
        const int e = V ? i / (4 * U) * U + i % U : i * 8 % D + j;
        const uint32_t q = (uint32_t)(code_of(h2f(b.x[t][e]), s, inv) + 128) & 255u;
        w[j >> 2] = (w[j >> 2] & ~(255u << (8 * (j & 3)))) | q << (8 * (j & 3));
      }
    }
    *reinterpret_cast<uint2*>(codes + (size_t)i * 8) = make_uint2(w[0], w[1]);
  }
  return s;
}

// One wave's share of an append: block `b` (0: the one that the tail began) of one head; for block 0 also what is left
// over as the new tail, so that the rows of the old one are read before the new ones are written. K and V one after
// the other through the wave's LDS.
template <int D>
__device__ void append_block(const Kv8Dev& c, const KvRows& k, const KvRows& v, int s, int sc, int h, int b, int n,
                             int len, BlockLds<D>& lds) {
  const int lane = threadIdx.x & 63;
  const int r = len % kKvBlock, whole = (r + n) / kKvBlock;
  const size_t head = (size_t)s * c.kvh + h;
  if (b >= whole && b > 0) return;
  int slot = 0;
  if (b < whole) slot = kv_slot(c, c.table[head * c.slots + len / kKvBlock + b]);
  uint32_t bad = whole ? 0u : c.bad[head];
#pragma unroll 1
  for (int p = 0; p < 2; p++) {
    const KvRows& in = p ? v : k;
    uint16_t* tail = (p ? c.vt : c.kt) + head * kKvBlock * D;
    const long long base = sc * in.seq + h * in.head;
    if (b < whole) {
      for (int i = lane; i < kKvBlock * D; i += 64) {
        const int t = i / D, e = i % D, row = b * kKvBlock - r + t;  // row of the call; below 0: of the tail
        lds.x[t][e] = row >= 0 ? row_elem(in, base + row * in.pos + e) : tail[p ? v_place<D>(t, e) : i];
      }
      wave_lds_sync();
      uint8_t* codes = (p ? c.vc : c.kc) + (head * c.slots + slot) * (size_t)(kKvBlock * D);
      const float sc2 = p ? code_block<D, true>(lds, lane, codes) : code_block<D, false>(lds, lane, codes);
      if (lane == 0) (p ? c.vs : c.ks)[head * c.slots + slot] = sc2;
      wave_lds_sync();
    }
    if (b == 0) {  // rows [t0, t1) of the tail that is there after the call
      const int t0 = whole ? 0 : r, t1 = whole ? (r + n) % kKvBlock : r + n;
      for (int t = t0; t < t1; t++) {
        const int row = whole * kKvBlock - r + t;
        bool off = false;
        for (int e = lane; e < D; e += 64) {
          const uint16_t x = row_elem(in, base + row * in.pos + e);
          tail[p ? v_place<D>(t, e) : t * D + e] = x;
          off |= (x & 0x7fff) >= 0x7c00;
        }
        bad = p == 0 ? bad & ~(1u << t) : bad;
        if (__ballot(off)) bad |= 1u << t;
      }
    }
  }
  if (b == 0 && lane == 0) c.bad[head] = bad;
}

// n = 1: a workgroup per sequence, its waves the heads; the length moves on behind the last of them.
template <int D>
__global__ __launch_bounds__(512) void k_kv8_append_one(Kv8Dev c, KvRows k, KvRows v, int seq0) {
  __shared__ BlockLds<D> lds[8];
  const int sc = blockIdx.x, s = seq0 + sc, w = threadIdx.x >> 6, W = blockDim.x >> 6;
  const int len = kv_len(c, s);
  if (len + 1 > c.max_len) {
    if (threadIdx.x == 0) c.state[(size_t)s * KV_STATE + KV_DROPPED] += 1;
    return;
  }
  for (int h = w; h < c.kvh; h += W) append_block<D>(c, k, v, s, sc, h, 0, 1, len, lds[w]);
  __syncthreads();
  if (threadIdx.x == 0) c.state[(size_t)s * KV_STATE + KV_LEN] = len + 1;
}

// n > 1: a wave per block and head; k_kv8_advance follows.
template <int D>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8Dev c, KvRows k, KvRows v, int seq0, int n, int blocks) {
  __shared__ BlockLds<D> lds[4];
  const int w = threadIdx.x >> 6;
  const long long u = (long long)blockIdx.x * 4 + w;
  const int b = (int)(u % blocks), h = (int)(u / blocks), sc = blockIdx.y;
  if (h >= c.kvh) return;
  const int len = kv_len(c, seq0 + sc);
  if (len + n > c.max_len) return;
  append_block<D>(c, k, v, seq0 + sc, sc, h, b, n, len, lds[w]);
}

__global__ void k_kv8_advance(Kv8Dev c, int seq0, int n_seqs, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_seqs) return;
  const int len = kv_len(c, seq0 + i);
  int* st = c.state + (size_t)(seq0 + i) * KV_STATE;
  if (len + n > c.max_len) st[KV_DROPPED] += n;
  else st[KV_LEN] = len + n;
}

__global__ void k_kv8_clear(Kv8Dev c, int seq0) {
  const int s = seq0 + blockIdx.y;
  const size_t head = (size_t)s * c.kvh;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < c.kvh * c.slots) {
    c.table[head * c.slots + i] = i % c.slots;
    if (c.mass) c.mass[head * c.slots + i] = 0.0f;
  }
  if (i < c.kvh) c.bad[head + i] = 0u;
  if (i < KV_STATE) c.state[(size_t)s * KV_STATE + i] = 0;
}

// A workgroup per block of the positions asked for (aligned as the call's, not as the cache's) and head.
template <int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Dev c, KvRows k, KvRows v, int seq0, int pos, int n) {
  const int sc = blockIdx.z, h = blockIdx.y, s = seq0 + sc, len = kv_len(c, s);
  const size_t head = (size_t)s * c.kvh + h;
  const int first = pos < 0 ? len + pos : pos;
  for (int i = threadIdx.x; i < kKvBlock * D; i += blockDim.x) {
    const int row = blockIdx.x * kKvBlock + i / D, e = i % D;
    if (row >= n) break;
    const int at = first + row, b = at / kKvBlock, t = at % kKvBlock;
    const bool in = at >= 0 && at < len, tail = in && b == len / kKvBlock;
    size_t slot = 0;
    if (in && !tail) slot = head * c.slots + kv_slot(c, c.table[head * c.slots + b]);
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const KvRows& out = p ? v : k;
      float x = 0.0f;
      if (in) {
        const int place = p ? v_place<D>(t, e) : t * D + e;
        if (tail) x = h2f((p ? c.vt : c.kt)[head * kKvBlock * D + place]);
        else x = (float)((int)(p ? c.vc : c.kc)[slot * (kKvBlock * D) + place] - 128) * (p ? c.vs : c.ks)[slot];
      }
      const long long o = sc * out.seq + row * out.pos + h * out.head + e;
      if (out.f16) ((uint16_t*)out.p)[o] = f2h(x);
      else ((float*)out.p)[o] = x;
    }
  }
}

// Order of masses as unsigned integers: numbers by value (-0 as 0), NaN above all.
__device__ __forceinline__ uint32_t mass_key(float m) {
  m = m + 0.0f;
  if (m != m) return 0xffffffffu;
  const uint32_t b = __float_as_uint(m);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kEvictThreads = 1024;

// Sum over the workgroup's threads before this one, and all of them.
__device__ int block_prefix(int v, int* waves, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[w] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < kEvictThreads / 64; i++) {
    before += i < w ? waves[i] : 0;
    all += waves[i];
  }
  *total = all;
  return before + x - v;
}

// A workgroup per head. Thread i holds blocks i KPT .. i KPT + KPT - 1 (their table entries and mass keys, in
// registers, so the table can be rewritten in place once all have been read). The key of the last block that stays is
// found 8 bits at a time by counting; among blocks of that key the earlier stay.
template <int KPT>
__global__ __launch_bounds__(kEvictThreads) void k_kv8_evict(Kv8Dev c, int seq0, int keep, int first, int last) {
  __shared__ int hist[256], waves[kEvictThreads / 64], pick[2];
  const int s = seq0 + blockIdx.x / c.kvh, len = kv_len(c, s), nb = len / kKvBlock;
  if (nb <= keep) return;
  const size_t base = ((size_t)s * c.kvh + blockIdx.x % c.kvh) * c.slots;
  const int i0 = threadIdx.x * KPT;
  int slot[KPT];
  uint32_t key[KPT];
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    const int i = i0 + j;
    slot[j] = i < nb ? c.table[base + i] : 0;
    key[j] = i >= first && i < nb - last ? mass_key(c.mass[base + kv_slot(c, slot[j])]) : 0u;
  }
  int left = keep - first - last;  // blocks that stay of those that may leave
  uint32_t pre = 0;                // bits of the key of the last that stays, from the top
  for (int sh = 24; sh >= 0 && left > 0; sh -= 8) {
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KPT; j++) {
      const int i = i0 + j;
      if (i >= first && i < nb - last && (sh == 24 || key[j] >> (sh + 8) == pre >> (sh + 8)))
        atomicAdd(&hist[key[j] >> sh & 255u], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int x = 255, above = 0;
      while (above + hist[x] < left) above += hist[x--];
      pick[0] = x;
      pick[1] = above;
    }
    __syncthreads();
    pre |= (uint32_t)pick[0] << sh;
    left -= pick[1];
  }
  // `left` blocks of key `pre` stay, and all above it
  bool may[KPT], stays[KPT];
  int same = 0, total;
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    may[j] = i0 + j >= first && i0 + j < nb - last;
    same += may[j] && left > 0 && key[j] == pre ? 1 : 0;
  }
  int before = block_prefix(same, waves, &total), stay = 0;
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    const bool eq = may[j] && left > 0 && key[j] == pre;
    stays[j] = i0 + j < nb && (!may[j] || (keep > first + last && key[j] > pre) || (eq && before < left));
    before += eq ? 1 : 0;
    stay += stays[j] ? 1 : 0;
  }
  int to = block_prefix(stay, waves, &total);
  const bool tail = len % kKvBlock != 0;
  const int tail_slot = tail && threadIdx.x == 0 ? c.table[base + nb] : 0;
  int gone = keep + (tail ? 1 : 0) + min(i0, nb) - to;  // place of this thread's first block that leaves
  __syncthreads();
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    if (i0 + j < nb) {
      c.table[base + (stays[j] ? to : gone)] = slot[j];
      if (!stays[j]) c.mass[base + kv_slot(c, slot[j])] = 0.0f;
    }
    to += stays[j] ? 1 : 0;
    gone += stays[j] ? 0 : 1;
  }
  if (tail && threadIdx.x == 0) c.table[base + keep] = tail_slot;
}

__global__ void k_kv8_shorten(Kv8Dev c, int seq0, int n_seqs, int keep) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_seqs) return;
  const int len = kv_len(c, seq0 + i);
  if (len / kKvBlock > keep) c.state[(size_t)(seq0 + i) * KV_STATE + KV_LEN] = keep * kKvBlock + len % kKvBlock;
}

}  // namespace

hipError_t launch_kv8_clear(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs) {
  klaunch(k_kv8_clear, dim3((c.kvh * c.slots + 255) / 256, n_seqs), 256, 0, s, c, seq0);
  return hipGetLastError();
}

hipError_t launch_kv8_append(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, KvRows k, KvRows v, int n) {
  if (n == 1) {
    const int threads = 64 * (c.kvh < 8 ? c.kvh : 8);
    if (c.d == 64) klaunch(k_kv8_append_one<64>, n_seqs, threads, 0, s, c, k, v, seq0);
    else klaunch(k_kv8_append_one<128>, n_seqs, threads, 0, s, c, k, v, seq0);
    return hipGetLastError();
  }
  const int blocks = (kKvBlock - 1 + n) / kKvBlock;
  const dim3 grid((unsigned)(((long long)blocks * c.kvh + 3) / 4), n_seqs);
  if (c.d == 64) klaunch(k_kv8_append<64>, grid, 256, 0, s, c, k, v, seq0, n, blocks);
  else klaunch(k_kv8_append<128>, grid, 256, 0, s, c, k, v, seq0, n, blocks);
  klaunch(k_kv8_advance, (n_seqs + 63) / 64, 64, 0, s, c, seq0, n_seqs, n);
  return hipGetLastError();
}

hipError_t launch_kv8_read(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int pos, int n, KvRows k, KvRows v) {
  const dim3 grid((n + kKvBlock - 1) / kKvBlock, c.kvh, n_seqs);
  if (c.d == 64) klaunch(k_kv8_read<64>, grid, 256, 0, s, c, k, v, seq0, pos, n);
  else klaunch(k_kv8_read<128>, grid, 256, 0, s, c, k, v, seq0, pos, n);
  return hipGetLastError();
}

hipError_t launch_kv8_evict(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int keep, int first, int last) {
  const int grid = n_seqs * c.kvh;
#define EVICT(K)                                                                               \
  if (c.slots <= K * kEvictThreads) {                                                          \
    klaunch(k_kv8_evict<K>, grid, kEvictThreads, 0, s, c, seq0, keep, first, last);            \
    klaunch(k_kv8_shorten, (n_seqs + 63) / 64, 64, 0, s, c, seq0, n_seqs, keep);               \
    return hipGetLastError();                                                                  \
  }
  EVICT(1) EVICT(2) EVICT(4) EVICT(8) EVICT(16) EVICT(32)
#undef EVICT
  return hipErrorInvalidValue;
}

}  // namespace moert

// ---- C entry points --------------------------------------------------------------------------------------------
using namespace moert;

namespace {

#define KV_CFG(cond, ...) \
  do {                    \
    if (!(cond)) return set_error(MOERT_E_CONFIG, __VA_ARGS__); \
  } while (0)

#define KV_HIP(expr)                                                                                            \
  do {                                                                                                          \
    const hipError_t e_ = (expr);                                                                               \
    if (e_ != hipSuccess)                                                                                       \
      return set_error(MOERT_E_DEVICE, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

#define KV_TRY(expr)             \
  do {                           \
    const int rc_ = (expr);      \
    if (rc_ != MOERT_OK) return rc_; \
  } while (0)

constexpr int kKvMaxLen = 1 << 20, kKvMaxSeqs = 65535, kKvMaxHeads = 256;

int view(const char* what, const moert_kv8* c, int seq0, int n_seqs, bool mass, Kv8Dev* d) {
  KV_CFG(c, "%s: null cache", what);
  KV_CFG(c->seqs >= 1 && c->seqs <= kKvMaxSeqs && c->kv_heads >= 1 && c->kv_heads <= kKvMaxHeads &&
             (c->head_dim == 64 || c->head_dim == 128) && c->max_len >= kKvBlock && c->max_len % kKvBlock == 0 &&
             c->max_len <= kKvMaxLen,
         "%s: %d sequences, %d KV heads of %d, max_len %d", what, c->seqs, c->kv_heads, c->head_dim, c->max_len);
  KV_CFG(c->k_codes_dev && c->v_codes_dev && c->k_scale_dev && c->v_scale_dev && c->k_tail_dev && c->v_tail_dev &&
             c->tail_bad_dev && c->table_dev && c->state_dev && (!mass || c->mass_dev),
         "%s: a null buffer", what);
  const uintptr_t wide = (uintptr_t)c->k_codes_dev | (uintptr_t)c->v_codes_dev | (uintptr_t)c->k_tail_dev |
                         (uintptr_t)c->v_tail_dev;
  const uintptr_t words = (uintptr_t)c->k_scale_dev | (uintptr_t)c->v_scale_dev | (uintptr_t)c->tail_bad_dev |
                          (uintptr_t)c->table_dev | (uintptr_t)c->mass_dev | (uintptr_t)c->state_dev;
  KV_CFG(wide % 16 == 0 && words % 4 == 0, "%s: codes and tails are aligned to 16 bytes, the others to 4", what);
  KV_CFG(seq0 >= 0 && n_seqs >= 1 && n_seqs <= c->seqs - seq0, "%s: sequences %d + %d of %d", what, seq0, n_seqs,
         c->seqs);
  *d = Kv8Dev{c->seqs,       c->kv_heads,   c->head_dim,   c->max_len / kKvBlock, c->max_len,
              c->k_codes_dev, c->v_codes_dev, c->k_scale_dev, c->v_scale_dev,       c->k_tail_dev,
              c->v_tail_dev,  c->tail_bad_dev, c->table_dev,  c->mass_dev,          c->state_dev};
  return MOERT_OK;
}

// Rows that a call reads or (out) writes.
int rows(const char* what, const moert_rows* r, int n_seqs, int n, int heads, int d, bool out, KvRows* k) {
  KV_CFG(r && r->data_dev, "%s: null rows", what);
  KV_CFG(r->dtype == MOERT_F32 || r->dtype == MOERT_F16, "%s: rows of dtype %d", what, r->dtype);
  KV_CFG((uintptr_t)r->data_dev % (r->dtype == MOERT_F32 ? 4 : 2) == 0, "%s: rows not aligned to their type", what);
  if (out) {
    // each axis, from the one with the least stride on, has to clear all that the ones before it span
    struct Axis {
      long long stride;
      int count;
    } a[3] = {{r->seq_stride, n_seqs}, {r->pos_stride, n}, {r->head_stride, heads}};
    for (int i = 0; i < 2; i++)
      for (int j = 0; j < 2 - i; j++)
        if (a[j].stride > a[j + 1].stride) {
          const Axis t = a[j];
          a[j] = a[j + 1];
          a[j + 1] = t;
        }
    __int128 span = d;
    for (const Axis& x : a)
      if (x.count > 1) {
        KV_CFG(x.stride >= span, "%s: rows to be written overlap (strides %lld, %lld, %lld)", what, r->seq_stride,
               r->pos_stride, r->head_stride);
        span += (__int128)x.stride * (x.count - 1);
      }
  }
  *k = KvRows{r->data_dev, r->dtype == MOERT_F16, r->seq_stride, r->pos_stride, r->head_stride};
  return MOERT_OK;
}

// Makes the buffers' device the current one while the call lasts.
class OnDevice {
 public:
  ~OnDevice() {
    if (back_ >= 0) (void)hipSetDevice(back_);
  }
  int enter(const char* what, const void* p) {
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
      (void)hipGetLastError();  // an address that the runtime does not know is no device error
      return set_error(MOERT_E_CONFIG, "%s: the cache is not in device memory", what);
    }
    KV_CFG(a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged, "%s: the cache is not in device memory",
           what);
    int now = -1;
    KV_HIP(hipGetDevice(&now));
    if (now != a.device) {
      KV_HIP(hipSetDevice(a.device));
      back_ = now;
    }
    return MOERT_OK;
  }

 private:
  int back_ = -1;
};

}  // namespace

extern "C" {

int moert_kv8_clear(const moert_kv8* c, int seq0, int n_seqs, void* stream) {
  Kv8Dev d;
  KV_TRY(view("kv8_clear", c, seq0, n_seqs, false, &d));
  OnDevice on;
  KV_TRY(on.enter("kv8_clear", d.kc));
  KV_HIP(launch_kv8_clear((hipStream_t)stream, d, seq0, n_seqs));
  return MOERT_OK;
}

int moert_kv8_append(const moert_kv8* c, int seq0, int n_seqs, const moert_rows* k, const moert_rows* v, int n,
                     void* stream) {
  Kv8Dev d;
  KvRows kr, vr;
  KV_TRY(view("kv8_append", c, seq0, n_seqs, false, &d));
  KV_CFG(n >= 1 && n <= d.max_len, "kv8_append: %d rows, max_len %d", n, d.max_len);
  KV_TRY(rows("kv8_append", k, n_seqs, n, d.kvh, d.d, false, &kr));
  KV_TRY(rows("kv8_append", v, n_seqs, n, d.kvh, d.d, false, &vr));
  OnDevice on;
  KV_TRY(on.enter("kv8_append", d.kc));
  KV_HIP(launch_kv8_append((hipStream_t)stream, d, seq0, n_seqs, kr, vr, n));
  return MOERT_OK;
}

int moert_kv8_read(const moert_kv8* c, int seq0, int n_seqs, int pos, int n, const moert_rows* k, const moert_rows* v,
                   void* stream) {
  Kv8Dev d;
  KvRows kr, vr;
  KV_TRY(view("kv8_read", c, seq0, n_seqs, false, &d));
  KV_CFG(n >= 1 && n <= d.max_len && pos >= -d.max_len && pos < d.max_len, "kv8_read: %d positions from %d, max_len %d",
         n, pos, d.max_len);
  KV_TRY(rows("kv8_read", k, n_seqs, n, d.kvh, d.d, true, &kr));
  KV_TRY(rows("kv8_read", v, n_seqs, n, d.kvh, d.d, true, &vr));
  OnDevice on;
  KV_TRY(on.enter("kv8_read", d.kc));
  KV_HIP(launch_kv8_read((hipStream_t)stream, d, seq0, n_seqs, pos, n, kr, vr));
  return MOERT_OK;
}

int moert_kv8_evict(const moert_kv8* c, int seq0, int n_seqs, int keep, int first, int last, void* stream) {
  Kv8Dev d;
  KV_TRY(view("kv8_evict", c, seq0, n_seqs, true, &d));
  KV_CFG(keep >= 0 && first >= 0 && last >= 0 && first <= keep && last <= keep - first,
         "kv8_evict: keep %d, first %d, last %d", keep, first, last);
  OnDevice on;
  KV_TRY(on.enter("kv8_evict", d.kc));
  KV_HIP(launch_kv8_evict((hipStream_t)stream, d, seq0, n_seqs, keep, first, last));
  return MOERT_OK;
}

static int attend_shape(const char* what, const Kv8Dev& d, int n_seqs, int heads, int n) {
  KV_CFG(heads >= 1 && heads % d.kvh == 0 && heads / d.kvh <= 64, "%s: %d query heads over %d KV heads", what, heads,
         d.kvh);
  KV_CFG(n >= 1 && n <= d.max_len, "%s: %d positions, max_len %d", what, n, d.max_len);
  KV_CFG((long long)n_seqs * heads * n <= 1 << 28, "%s: %d sequences x %d positions x %d heads", what, n_seqs, n, heads);
  return MOERT_OK;
}

int moert_kv8_workspace(const moert_kv8* c, int n_seqs, int heads, int n, int track, size_t* bytes) {
  Kv8Dev d;
  KV_TRY(view("kv8_workspace", c, 0, n_seqs, false, &d));
  KV_CFG(bytes, "kv8_workspace: null bytes");
  KV_TRY(attend_shape("kv8_workspace", d, n_seqs, heads, n));
  *bytes = kv8_attn_plan(d, n_seqs, heads, n, track != 0).bytes;
  return MOERT_OK;
}

int moert_kv8_attend(const moert_kv8* c, int seq0, int n_seqs, int heads, int n, float scale, const moert_rows* q,
                     const moert_rows* out, float mass_decay, void* ws_dev, size_t ws_bytes, void* stream) {
  Kv8Dev d;
  KvRows qr, orow;
  KV_CFG(mass_decay <= 1.0f, "kv8_attend: mass_decay %g", (double)mass_decay);  // NaN among the refused
  const bool track = mass_decay >= 0.0f;
  KV_TRY(view("kv8_attend", c, seq0, n_seqs, track, &d));
  KV_TRY(attend_shape("kv8_attend", d, n_seqs, heads, n));
  KV_CFG(scale - scale == 0.0f, "kv8_attend: scale %g", (double)scale);
  KV_TRY(rows("kv8_attend", q, n_seqs, n, heads, d.d, false, &qr));
  KV_TRY(rows("kv8_attend", out, n_seqs, n, heads, d.d, true, &orow));
  KV_CFG(q->dtype == out->dtype, "kv8_attend: q of dtype %d, out of %d", q->dtype, out->dtype);
  const KvAttnPlan p = kv8_attn_plan(d, n_seqs, heads, n, track);
  KV_CFG(ws_dev && (uintptr_t)ws_dev % 16 == 0 && ws_bytes >= p.bytes,
         "kv8_attend: a workspace of %zu bytes aligned to 16 is needed, got %zu", p.bytes, ws_bytes);
  OnDevice on;
  KV_TRY(on.enter("kv8_attend", d.kc));
  KV_HIP(launch_kv8_attend((hipStream_t)stream, d, seq0, n_seqs, heads, n, scale, qr, orow, mass_decay, ws_dev));
  return MOERT_OK;
}

int moert_kv8_lengths(const moert_kv8* c, int seq0, int n_seqs, int* lengths, void* stream) {
  Kv8Dev d;
  KV_TRY(view("kv8_lengths", c, seq0, n_seqs, false, &d));
  KV_CFG(lengths, "kv8_lengths: null lengths");
  OnDevice on;
  KV_TRY(on.enter("kv8_lengths", d.kc));
  hipStream_t s = (hipStream_t)stream;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  KV_HIP(hipStreamIsCapturing(s, &cs));
  KV_CFG(cs == hipStreamCaptureStatusNone, "kv8_lengths: the stream is being captured");
  int dropped = 0, part[64 * KV_STATE];
  for (int i = 0; i < n_seqs; i += 64) {
    const int m = n_seqs - i < 64 ? n_seqs - i : 64;
    KV_HIP(hipMemcpyAsync(part, d.state + (size_t)(seq0 + i) * KV_STATE, (size_t)m * KV_STATE * 4,
                          hipMemcpyDeviceToHost, s));
    KV_HIP(hipStreamSynchronize(s));
    for (int j = 0; j < m; j++) {
      lengths[i + j] = part[j * KV_STATE + KV_LEN];
      if (part[j * KV_STATE + KV_DROPPED] && !dropped) dropped = 1 + i + j;
    }
  }
  if (dropped)
    return set_error(MOERT_E_FULL, "kv8_lengths: sequence %d has dropped rows for want of room", seq0 + dropped - 1);
  return MOERT_OK;
}

}  // extern "C"
