// The 8-bit K/V cache: append, read back, eviction, and the C entry points (kv8_attn.hip has the attention).
#include "kv8.h"

#include "../../include/moert.h"
#include "launch.h"
#include "rows_api.h"

namespace moert {

namespace {

// Eight elements of a row as fp16 bits. vec: the rows' strides and pointer allow 16-byte loads.
__device__ __forceinline__ uint4 row_halves(const KvRows& r, long long at, bool vec) {
  uint32_t w[4];
  if (r.f16) {
    const uint16_t* p = (const uint16_t*)r.p + at;
    if (vec) return gload_u4(p);
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)gmem(p)[2 * i] | (uint32_t)gmem(p)[2 * i + 1] << 16;
  } else {
    const float* p = (const float*)r.p + at;
    float x[8];
    if (vec) {
      const float4 a = gload_f4(p), b = gload_f4(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = gmem(p)[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// round(x / s) + 128 of eight fp16 as bytes, ties to even, of the exact quotients. q = round(x * inv) is off by less
// than one, next to a tie; there the residual x - q s (one fma) is a multiple of ulp(s) / 2 below s, so it is exact and
// tells: below s / 2, q is right, and that is all that nearly every wave has to look at.
__device__ __forceinline__ uint2 codes_of(const uint16_t* x, float s, float inv) {
  const float h = 0.5f * s;
  float q[8], r[8], most = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    q[i] = __builtin_rintf(h2f(x[i]) * inv);
    r[i] = __builtin_fmaf(-q[i], s, h2f(x[i]));
    most = __builtin_fmaxf(most, __builtin_fabsf(r[i]));
  }
  if (__any(most >= h)) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float d = __builtin_fabsf(r[i]);
      q[i] += d > h || (d == h && ((int)q[i] & 1)) ? __builtin_copysignf(1.0f, r[i]) : 0.0f;
    }
  }
  uint32_t o[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; i++) o[i >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(q[i] + 128.0f, i & 3, o[i >> 2]);
  return make_uint2(o[0], o[1]);
}

// Largest magnitude of eight fp16, as bits.
__device__ __forceinline__ int top_of(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  int m = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) m = max(m, max((int)(w[i] & 0x7fffu), (int)(w[i] >> 16 & 0x7fffu)));
  return m;
}

// Counts rows that found no room, up to the type's largest number: no count of them comes back to 0, which is none.
__device__ __forceinline__ void count_dropped(int* state, int n) {
  const int had = state[KV_DROPPED];
  state[KV_DROPPED] = had > 0x7fffffff - n ? 0x7fffffff : had + n;
}

constexpr int kAppendThreads = 256;

// A workgroup per block and KV head: its first half codes K, the other V, 8 elements of a row to a thread at a time, in
// registers (bound by memory: 16391 rows of two sequences, 100 MB, in 28.5 us; a wave per block, element by element,
// took 102). V goes through LDS to its own order. The workgroup of block 0, the one that the old tail began, also
// writes the new tail, once the old one's rows have been read. arrive: the last workgroup of a sequence to get there
// moves its length on, where few do (the counter's additions come one after the other: 8208 workgroups took 100 us);
// otherwise k_kv8_advance does.
template <int D>
__global__ __launch_bounds__(kAppendThreads) void k_kv8_append(Kv8Dev c, KvRows k, KvRows v, int seq0, int n,
                                                               int blocks, int vec, int arrive) {
  constexpr int C = D / 32, R = D / 8, U = D / 16;  // a thread's chunks of 8, a row's, elements of a run of V
  __shared__ __align__(16) uint16_t lds[kKvBlock][D + 8];
  __shared__ int tops[4];
  __shared__ uint32_t bad_rows;
  const int b = blockIdx.x % blocks, h = blockIdx.x / blocks, sc = blockIdx.y, s = seq0 + sc;
  const int p = threadIdx.x >> 7, x = threadIdx.x & 127;
  const int len = kv_len(c, s);
  int* state = c.state + (size_t)s * KV_STATE;
  if (len + n > c.max_len) {
    if (arrive && blockIdx.x == 0 && threadIdx.x == 0) count_dropped(state, n);
    return;
  }
  const int r = len % kKvBlock, whole = (r + n) / kKvBlock;
  const size_t head = (size_t)s * c.kvh + h;
  const KvRows in = p ? v : k;
  const bool wide = vec >> p & 1;
  uint16_t* tail = (p ? c.vt : c.kt) + head * kKvBlock * D;
  const long long base = sc * in.seq + h * in.head;
  if (b < whole) {
    const size_t slot = head * c.slots + kv_slot(c, c.table[head * c.slots + len / kKvBlock + b]);
    uint4 q[C];
    int top = 0;
#pragma unroll
    for (int j = 0; j < C; j++) {
      const int t = (x + 128 * j) / R, e = (x + 128 * j) % R * 8, row = b * kKvBlock - r + t;
      if (row >= 0) q[j] = row_halves(in, base + row * in.pos + e, wide);
      else if (p == 0) q[j] = gload_u4(tail + t * D + e);
      else continue;
      top = max(top, top_of(q[j]));
      if (p) *reinterpret_cast<uint4*>(&lds[t][e]) = q[j];
    }
    if (p && b == 0 && r) {  // V's old tail, a run of 8 positions of an element at a time
#pragma unroll
      for (int j = 0; j < C; j++) {
        const int i = x + 128 * j, t = i / U % 4 * 4, e = i / (4 * U) * U + i % U;
        const uint4 y = gload_u4(tail + i * 8);
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int z = 0; z < 8; z++) {
          const int tz = t + (z & 3) + 16 * (z >> 2);
          const uint16_t a = (uint16_t)(w[z >> 1] >> (16 * (z & 1)));
          if (tz < r) {
            lds[tz][e] = a;
            top = max(top, a & 0x7fff);
          }
        }
      }
    }
    top = max(top, partner<1>(top));
    top = max(top, partner<2>(top));
    top = max(top, partner<4>(top));
    top = max(top, partner<8>(top));
    top = max(top, partner<16>(top));
    top = max(top, partner<32>(top));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(tops[2 * p], tops[2 * p + 1]);
    const bool bad = top >= 0x7c00;
    const float sc8 = top && !bad ? h2f((uint16_t)top) / 127.0f : 1.0f, inv = 1.0f / sc8;
    uint8_t* codes = (p ? c.vc : c.kc) + slot * (size_t)(kKvBlock * D);
#pragma unroll
    for (int j = 0; j < C; j++) {
      const int i = x + 128 * j;
      const uint32_t w[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
      uint16_t a[8];
#pragma unroll
      for (int y = 0; y < 8; y++)  // V: run i is ((element / U) * 4 + group) * U + element % U
        a[y] = p ? lds[i / U % 4 * 4 + (y & 3) + 16 * (y >> 2)][i / (4 * U) * U + i % U]
                 : (uint16_t)(w[y >> 1] >> (16 * (y & 1)));
      const uint2 o = codes_of(a, sc8, inv);
      *reinterpret_cast<uint2*>(codes + i * 8) = bad ? make_uint2(0x80808080u, 0x80808080u) : o;
    }
    if (x == 0) (p ? c.vs : c.ks)[slot] = bad ? __int_as_float(0x7fc00000) : sc8;
  }
  if (b == 0) {  // rows [t0, t1) of the tail that is there after the call
    const int t0 = whole ? 0 : r, t1 = whole ? (r + n) % kKvBlock : r + n;
    if (threadIdx.x == 0) bad_rows = 0u;
    __syncthreads();
    for (int i = x; i < (t1 - t0) * R; i += 128) {
      const int t = t0 + i / R, e = i % R * 8, row = whole * kKvBlock - r + t;
      const uint4 y = row_halves(in, base + row * in.pos + e, wide);
      if (p == 0) {
        *reinterpret_cast<uint4*>(tail + t * D + e) = y;
      } else {
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int z = 0; z < 8; z++) tail[v_place<D>(t, e + z)] = (uint16_t)(w[z >> 1] >> (16 * (z & 1)));
      }
      if (top_of(y) >= 0x7c00) atomicOr(&bad_rows, 1u << t);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t before = whole ? 0u : c.bad[head] & ((1u << r) - 1u);
      c.bad[head] = before | bad_rows;
    }
  }
  if (arrive) {
    __syncthreads();  // every wave has read the length
    if (threadIdx.x == 0 && atomicAdd(&state[KV_ARRIVED], 1) == (int)gridDim.x - 1) {
      state[KV_LEN] = len + n;
      state[KV_ARRIVED] = 0;
    }
  }
}

__global__ void k_kv8_advance(Kv8Dev c, int seq0, int n_seqs, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_seqs) return;
  const int len = kv_len(c, seq0 + i);
  int* st = c.state + (size_t)(seq0 + i) * KV_STATE;
  if (len + n > c.max_len) count_dropped(st, n);
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

// A workgroup per block of the cache and head, its first half K, the other V; the codes go through LDS, where V comes
// back to rows, and out 8 elements of a row at a time (100 MB in 22 us; byte by byte without LDS 55). Positions that
// are not there give 0: their blocks lie before the sequence's first one or behind its last.
template <int D>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Dev c, KvRows k, KvRows v, int seq0, int pos, int n, int vec) {
  constexpr int C = D / 32, R = D / 8, U = D / 16;
  __shared__ __align__(16) float lds[2][kKvBlock][D + 4];
  const int sc = blockIdx.z, h = blockIdx.y, s = seq0 + sc, len = kv_len(c, s);
  const size_t head = (size_t)s * c.kvh + h;
  const int first = pos < 0 ? len + pos : pos;           // position of the call's row 0
  const int b = (first - (first & 31)) / kKvBlock + (int)blockIdx.x;  // whole numbers below 0 too
  const int p = threadIdx.x >> 7, x = threadIdx.x & 127;
  const bool tail = b == len / kKvBlock, in = b >= 0 && b * kKvBlock < len;
  if (in && !tail) {
    const size_t slot = head * c.slots + kv_slot(c, c.table[head * c.slots + b]);
    const float sc8 = (p ? c.vs : c.ks)[slot];
    const uint8_t* codes = (p ? c.vc : c.kc) + slot * (size_t)(kKvBlock * D);
#pragma unroll
    for (int j = 0; j < C; j++) {
      const int i = x + 128 * j;
      const uint2 w = gload_u2(codes + i * 8);
#pragma unroll
      for (int y = 0; y < 8; y++) {
        const float z = (float)((int)((y < 4 ? w.x : w.y) >> (8 * (y & 3)) & 255u) - 128) * sc8;
        if (p) lds[1][i / U % 4 * 4 + (y & 3) + 16 * (y >> 2)][i / (4 * U) * U + i % U] = z;
        else lds[0][i / R][i % R * 8 + y] = z;
      }
    }
  } else if (in) {
    const uint16_t* t16 = (p ? c.vt : c.kt) + head * kKvBlock * D;
#pragma unroll
    for (int j = 0; j < C; j++) {
      const int i = x + 128 * j;
      const uint4 q = gload_u4(t16 + i * 8);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int y = 0; y < 8; y++) {
        const float z = h2f((uint16_t)(w[y >> 1] >> (16 * (y & 1))));
        if (p) lds[1][i / U % 4 * 4 + (y & 3) + 16 * (y >> 2)][i / (4 * U) * U + i % U] = z;
        else lds[0][i / R][i % R * 8 + y] = z;
      }
    }
  }
  __syncthreads();
  const KvRows out = p ? v : k;
#pragma unroll
  for (int j = 0; j < C; j++) {
    const int t = (x + 128 * j) / R, e = (x + 128 * j) % R * 8, at = b * kKvBlock + t, row = at - first;
    if (row < 0 || row >= n) continue;
    const bool there = at >= 0 && at < len;
    float y[8];
#pragma unroll
    for (int z = 0; z < 8; z++) y[z] = there ? lds[p][t][e + z] : 0.0f;
    const long long o = sc * out.seq + row * out.pos + h * out.head + e;
    if (out.f16) {
      uint16_t* d = (uint16_t*)out.p + o;
      uint32_t w[4];
#pragma unroll
      for (int z = 0; z < 4; z++) w[z] = (uint32_t)f2h(y[2 * z]) | (uint32_t)f2h(y[2 * z + 1]) << 16;
      if (vec >> p & 1) {
        *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int z = 0; z < 8; z++) d[z] = (uint16_t)(w[z >> 1] >> (16 * (z & 1)));
      }
    } else {
      float* d = (float*)out.p + o;
      if (vec >> p & 1) {
        *reinterpret_cast<float4*>(d) = make_float4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<float4*>(d + 4) = make_float4(y[4], y[5], y[6], y[7]);
      } else {
#pragma unroll
        for (int z = 0; z < 8; z++) d[z] = y[z];
      }
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

// Sum over the workgroup's T threads before this one, and all of them.
template <int T>
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
#pragma unroll
  for (int i = 0; i < T / 64; i++) {
    before += i < w ? waves[i] : 0;
    all += waves[i];
  }
  *total = all;
  return before + x - v;
}

// A workgroup per head. Thread i holds blocks i KPT .. i KPT + KPT - 1 (their table entries and mass keys, in
// registers, so the table can be rewritten in place once all have been read). The key of the last block that stays is
// found by counting, 11, 11 and 10 bits at a time (the first take masses apart by a fifth, so that few counts meet in
// one bin: 13.8 us with 8 bits four times, 12.1 so, 4062 blocks of 128 heads); among blocks of that key the earlier stay.
template <int T, int KPT>
__global__ __launch_bounds__(T) void k_kv8_evict(Kv8Dev c, int seq0, int keep, int first, int last) {
  __shared__ __align__(16) int hist[2048];
  constexpr int B = 2048 / T;  // bins of a thread
  __shared__ int waves[T / 64], pick[2];
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
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    if (left <= 0) break;  // the same for all
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
#pragma unroll
    for (int j = 0; j < B; j++) hist[threadIdx.x + j * T] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KPT; j++) {
      const int i = i0 + j;
      if (i >= first && i < nb - last && (pass == 0 || (key[j] ^ pre) >> (sh + (pass == 1 ? 11 : 10)) == 0))
        atomicAdd(&hist[key[j] >> sh & (bins - 1)], 1);
    }
    __syncthreads();
    const int top = 2047 - B * (int)threadIdx.x;  // this thread's bins: top and the B - 1 below
    int v[B], mine = 0, total;
#pragma unroll
    for (int j = 0; j < B; j++) mine += v[j] = hist[top - j];
    int above = block_prefix<T>(mine, waves, &total);  // keys in the bins above them
#pragma unroll
    for (int j = 0; j < B; j++) {
      if (above < left && above + v[j] >= left) pick[0] = top - j, pick[1] = above;
      above += v[j];
    }
    __syncthreads();
    pre |= (uint32_t)pick[0] << sh;
    left -= pick[1];
  }
  // `left` blocks of key `pre` stay, and all above it
  bool may[KPT], stays[KPT];
  int same = 0;
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    may[j] = i0 + j >= first && i0 + j < nb - last;
    same += may[j] && left > 0 && key[j] == pre ? 1 : 0;
  }
  int total, before = block_prefix<T>(same, waves, &total), stay = 0;
#pragma unroll
  for (int j = 0; j < KPT; j++) {
    const bool eq = may[j] && left > 0 && key[j] == pre;
    stays[j] = i0 + j < nb && (!may[j] || (keep > first + last && key[j] > pre) || (eq && before < left));
    before += eq ? 1 : 0;
    stay += stays[j] ? 1 : 0;
  }
  int to = block_prefix<T>(stay, waves, &total);
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
  if (threadIdx.x == 0) {
    if (tail) c.table[base + keep] = tail_slot;
    int* state = c.state + (size_t)s * KV_STATE;  // every thread has read the length: the last head shortens it
    if (atomicAdd(&state[KV_ARRIVED], 1) == c.kvh - 1) {
      state[KV_LEN] = keep * kKvBlock + len % kKvBlock;
      state[KV_ARRIVED] = 0;
    }
  }
}

}  // namespace

hipError_t launch_kv8_clear(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs) {
  klaunch(k_kv8_clear, dim3((c.kvh * c.slots + 255) / 256, n_seqs), 256, 0, s, c, seq0);
  return hipGetLastError();
}

hipError_t launch_kv8_append(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, KvRows k, KvRows v, int n) {
  const int blocks = (kKvBlock - 1 + n) / kKvBlock, vec = wide_rows(k) | wide_rows(v) << 1;
  const int arrive = blocks * c.kvh <= 256;
  const dim3 grid(blocks * c.kvh, n_seqs);
  if (c.d == 64) klaunch(k_kv8_append<64>, grid, kAppendThreads, 0, s, c, k, v, seq0, n, blocks, vec, arrive);
  else klaunch(k_kv8_append<128>, grid, kAppendThreads, 0, s, c, k, v, seq0, n, blocks, vec, arrive);
  if (const hipError_t e = hipGetLastError()) return e;  // no rows, no length
  if (!arrive) klaunch(k_kv8_advance, (n_seqs + 63) / 64, 64, 0, s, c, seq0, n_seqs, n);
  return hipGetLastError();
}

hipError_t launch_kv8_read(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int pos, int n, KvRows k, KvRows v) {
  const dim3 grid((n + 2 * kKvBlock - 2) / kKvBlock, c.kvh, n_seqs);
  const int vec = wide_rows(k) | wide_rows(v) << 1;
  if (c.d == 64) klaunch(k_kv8_read<64>, grid, 256, 0, s, c, k, v, seq0, pos, n, vec);
  else klaunch(k_kv8_read<128>, grid, 256, 0, s, c, k, v, seq0, pos, n, vec);
  return hipGetLastError();
}

hipError_t launch_kv8_evict(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int keep, int first, int last) {
  const int grid = n_seqs * c.kvh;
  // Short tables take fewer threads, whose barriers cost less (7.7 us for 8.7 with 1024, 144 slots, 7.9 for 8.9 with 512);
  // long ones as many as there are: fewer, with more keys each, are slower (130000 positions: 14.2 us, 15.8 with 512).
#define EVICT(T, K)                                                        \
  if (c.slots <= K * T) {                                                  \
    klaunch(k_kv8_evict<T, K>, grid, T, 0, s, c, seq0, keep, first, last); \
    return hipGetLastError();                                              \
  }
  EVICT(256, 1) EVICT(512, 1) EVICT(1024, 1) EVICT(1024, 2) EVICT(1024, 4) EVICT(1024, 8) EVICT(1024, 16) EVICT(1024, 32)
#undef EVICT
  return hipErrorInvalidValue;
}

}  // namespace moert

// ---- C entry points --------------------------------------------------------------------------------------------
using namespace moert;

namespace {

constexpr int kOf8Bits = 1 << MOERT_F32 | 1 << MOERT_F16;
constexpr int kKvMaxLen = 1 << 20, kKvMaxSeqs = 65535, kKvMaxHeads = 256;

int view(const char* what, const moert_kv8* c, int seq0, int n_seqs, bool mass, Kv8Dev* d) {
  KV_CFG(c, "%s: null cache", what);
  KV_CFG(c->seqs >= 1 && c->seqs <= kKvMaxSeqs && c->kv_heads >= 1 && c->kv_heads <= kKvMaxHeads &&
             (long long)c->seqs * c->kv_heads <= 1 << 20 && (c->head_dim == 64 || c->head_dim == 128) &&
             c->max_len >= kKvBlock && c->max_len % kKvBlock == 0 &&
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
  KV_TRY(rows("kv8_append", k, kOf8Bits, n_seqs, n, d.kvh, d.d, false, &kr));
  KV_TRY(rows("kv8_append", v, kOf8Bits, n_seqs, n, d.kvh, d.d, false, &vr));
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
  KV_TRY(rows("kv8_read", k, kOf8Bits, n_seqs, n, d.kvh, d.d, true, &kr));
  KV_TRY(rows("kv8_read", v, kOf8Bits, n_seqs, n, d.kvh, d.d, true, &vr));
  KV_CFG(k->data_dev != v->data_dev, "kv8_read: K and V to one address");
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
  KV_CFG((long long)n_seqs * heads * n <= 1 << 27, "%s: %d sequences x %d positions x %d heads", what, n_seqs, n, heads);
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
  KV_TRY(rows("kv8_attend", q, kOf8Bits, n_seqs, n, heads, d.d, false, &qr));
  KV_TRY(rows("kv8_attend", out, kOf8Bits, n_seqs, n, heads, d.d, true, &orow));
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
