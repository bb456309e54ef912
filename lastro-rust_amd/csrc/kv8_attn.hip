// Attention over the 8-bit K/V cache (kv8.h), on the f16 matrix cores with f32 sums.
//
// A column is one query head at one position; the columns of a KV head, position by position, go in tiles of 16, NT of
// them to a wave. Per block of 32 positions of the cache:
//   S = K Q^T    MFMA 16x16x32, rows = 16 positions, columns = 16 columns. Codes become fp16 exactly (two bytes become
//                1024 + byte by one byte permutation, one packed subtraction takes 1152 off). A lane of group
//                G = lane / 16 reads 16 bytes of K row lane % 16, from element 16 G on.
//   softmax      u = s scale log2 e in base 2; the running maximum M of u + log2(scale of V) moves only when it has to
//                (by more than 8), so most blocks cost no exchange between lanes. p = 2^(u + log2 vs - M + 7): the
//                weights that meet the V codes carry the scale of V, so blocks of any scale add up in one accumulator,
//                and the largest contribution lies between 2^7 and 2^15, where fp16 has 11 bits down to 2^-21 of it and
//                stops at 2^-32. The sum of softmax and the blocks' weights take p / vs in f32, before p is rounded.
//                A block whose scale of V lies more than 2^8 below that of one that has moved M (zeros have scale 1)
//                would have its p below that, however much softmax weight it has: its p, and O for the time of its
//                products, are taken 2^k2 times as large, which brings its largest p to 2^6 or above. So the rounding
//                of a weight is off by its last bit or by 2^-24 of the column's largest weight. Beyond 2^16, where u
//                in f32 rounds the scales away, M follows u alone and every block is taken so: equal scores stay equal
//                weights, and no p leaves fp16 (M and the scales in one sum made it 2^17 and more from u of 2^24 on).
//   O += V^T P^T MFMA 16x16x32 over the 32 positions: rows = 16 elements, columns = columns. A lane of the S product
//                holds positions 4 G .. 4 G + 3 of both halves of the block for its column, which is what it has to
//                hold of P here when the positions of V are taken in that order: v_place lays V out so, and p never
//                leaves its lane.
// f32 queries enter as two fp16 (their row scaled by a power of two to below 2^10). p is taken as two fp16 for f32 outputs,
// and for fp16 ones of a single tile, where that is free (a pass over 131000 positions 33.8 us, over eight sequences 125,
// as with one) and brings them from 2.2-2.4e-4 off to the 2.0-2.2e-4 of their own rounding. Wider ones round p once: bound
// by the vector unit, 1000 positions after 16001 would take 242 us for 192, to be 2.1e-4 off for 2.4e-4.
//
// The waves of a workgroup take the blocks of their tile in turn and join in LDS; where the tiles are too few for the
// device, several workgroups share a tile (splits) and a second launch joins them. For eviction each block's sum goes
// out as log2 by column, which needs no final maximum, and a pass over them adds up the weights in a fixed order.
//
// What bounds it, measured on one MI355X (3B shape: 8 KV heads of 64, 3 query heads each):
//   one position   the cache's bytes: 134 MB of one sequence in 26 us (5.2 TB/s), 565 MB of eight in 110 us (5.2; blocks
//                  in any order; a streaming read of 512 MiB reaches 5.7). Short caches: launches (5.6 us for 100 rows).
//   many           the vector unit: 1000 positions after 16001, 101 GFLOP, in about 172 us in fp16. A block of two tiles
//                  is 16 MFMAs of 16 cycles beside 174 vector instructions, 64 of them the conversion of the codes, 16
//                  exps at a quarter of the rate; the vector unit issues in 83% of the time, the matrix cores are busy
//                  in 25%, 2.4 waves are on a SIMD. The whole pass is 192 us, with one tile to a wave 311; with 2 or 8
//                  waves to a workgroup 266 or 215 (131000 positions of one sequence, one each: 40 or 43 for 34);
//                  without the matrix instructions first (s_setprio) 195.5.
#include <math.h>

#include <type_traits>

#include "kv8.h"
#include "launch.h"

namespace moert {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kWaves = 4;       // waves of a workgroup, each its share of the blocks
constexpr int kMaxSplits = 64;  // one lane each in the combine
constexpr float kShift = 7.0f, kSlack = 8.0f;
constexpr float kApart = 8.0f;    // log2 of how far a block's scale of V may lie below one that M follows
constexpr float kFarL = 9.0f - kShift;  // L beside scores beyond 2^16: no scale of V is above 2^9.02 (65504 / 127)
constexpr float kMostUp = 60.0f;  // O is a sum of at most 2^20 products below 2^22, so it stays in range 2^60 times
constexpr float kNone = -3.4e38f;  // maximum of what has no score yet; finite, so that differences with it are

// a + the value of a's lane 16 (32) away, in both of them.
__device__ __forceinline__ float add16(float a) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Lanes 0 .. 31: a + a's lane 32 on; lanes 32 .. 63: the same of b.
__device__ __forceinline__ float add32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Eight codes + 128 as fp16: 0x64bb is 1024 + bb.
__device__ __forceinline__ h8 half_codes(uint32_t a, uint32_t b) {
  union {
    uint32_t w[4];
    h2 x[4];
    h8 v;
  } r;
  r.w[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  r.w[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  r.w[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  r.w[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
  for (int i = 0; i < 4; i++) r.x[i] -= off;
  return r.v;
}

// Eight elements of a row. wide: the rows' pointer and strides allow 16-byte loads.
template <bool F16>
__device__ __forceinline__ void load8(const KvRows& r, long long at, bool wide, float* x) {
  if constexpr (F16) {
    const uint16_t* p = (const uint16_t*)r.p + at;
    if (wide) {
      const uint4 v = gload_u4(p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = h2f((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = h2f(gmem(p)[j]);
    }
  } else {
    const float* p = (const float*)r.p + at;
    if (wide) {
      const float4 u = gload_f4(p), v = gload_f4(p + 4);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = gmem(p)[j];
    }
  }
}

// An output is a mean of values of at most 65504. Weights rounded to fp16 beside a sum that is not make it up to 2^-11
// more, and fp16 would have no number for it.
__device__ __forceinline__ float in_f16(float x) { return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x; }

// N elements (a multiple of 4) of a row of the output.
template <int N, bool F16>
__device__ __forceinline__ void store_out(const KvRows& r, long long at, bool wide, const float* x) {
  if constexpr (F16) {
    uint16_t* p = (uint16_t*)r.p + at;
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; j++) w[j] = (uint32_t)f2h(x[2 * j]) | (uint32_t)f2h(x[2 * j + 1]) << 16;
    if (wide) {
#pragma unroll
      for (int j = 0; j < N / 4; j++) *reinterpret_cast<uint2*>(p + 4 * j) = make_uint2(w[2 * j], w[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) p[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  } else {
    float* p = (float*)r.p + at;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      if (wide) *reinterpret_cast<f4*>(p + j) = f4{x[j], x[j + 1], x[j + 2], x[j + 3]};
      else p[j] = x[j], p[j + 1] = x[j + 1], p[j + 2] = x[j + 2], p[j + 3] = x[j + 3];
    }
  }
}

// Blocks that a column tile's last position sees, and the splits of it that have any: split x's waves take blocks
// x kWaves + wave, then every (splits kWaves)-th, so where a wave begins does not wait for the length.
__device__ __forceinline__ int blocks_seen(int len, int n, int g, int tile, int width) {
  const int last = min((tile + 1) * width - 1, n * g - 1) / g;  // last position of the tile
  return (max(0, len - n + 1 + last) + kKvBlock - 1) / kKvBlock;
}
__device__ __forceinline__ int splits_used(int blocks, int splits) {
  return max(1, min(splits, (blocks + kWaves - 1) / kWaves));
}

struct AttnArgs {
  Kv8Dev c;
  KvRows q, out;
  int seq0, n_seqs, g, n, splits, tiles;
  int vec;        // bit 0: q can be loaded 16 bytes at a time, bit 1: out can be stored so
  float kf;       // |scale| log2 e, less 2^ke
  int ke;
  uint32_t sign;  // of the scale
  float* part;    // [sequence, KV head, column][split][D]
  float2* ml;     // [sequence, KV head, column][split]: M + L, sum
  float* tot;     // [sequence, KV head, column]: log2 of the whole sum, +inf where nothing is seen
  float* lse;     // [sequence, KV head][block][column]: log2 of the block's sum
};

// log2 of a column's whole sum; +inf, which no weight survives, where it sees nothing. (A sum of 0 of rows that are
// seen, scores beyond f32, becomes NaN here and in the output.)
__device__ __forceinline__ float total_of(float m, float sum, bool none) {
  return none ? __int_as_float(0x7f800000) : __builtin_amdgcn_logf(sum) + m;
}
__device__ __forceinline__ bool sees_none(int len, int n, int g, int col) { return len - n + 1 + col / g <= 0; }

// STREAM: the codes are loaded with the non-temporal hint.
template <int D, bool F16, int NT, bool TRACK, bool STREAM>
__global__ __launch_bounds__(kWaves * 64, NT == 1 && D == 64 ? 4 : 2) void k_kv8_attend(AttnArgs a) {
  constexpr int KS = D / 32, U = D / 16, CH = D / 64, W = 16 * NT;
  constexpr bool LO = !F16 || NT == 1;  // p as two fp16
  // Which 16 elements a product of V has as its rows is free. A load of 16 bytes a lane takes 1 KB of V in a row, whole
  // cache lines: RP of the runs' rows, U / 2 pieces of each. (Two loads that each took half of every line asked the L2
  // for 1.8 times the bytes: 115 us where this takes 108, 565 MB.) So row i of product u is element elem(u, i).
  constexpr int RP = 16 / (U / 2);
  auto elem = [](int u, int i) { return (u / 2 * RP + i % RP) * U + 2 * (i / RP) + u % 2; };
  // blocks in flight: with two tiles, or the 8 KB blocks of wide heads, the other waves cover the loads (with two: sixteen
  // sequences of wide heads 34.5 us a pass for 32.6, one of 30000 positions 22.0 for 20.2; narrow ones gain with two where
  // waves are few: 131000 positions of one sequence 33.7 for 34.0 with one, of eight 124.8 for 123.1)
  constexpr int PF = NT == 1 && D == 64 ? 2 : 1;
  // One block in flight: the next one's K is asked for once this one's scores are there, not behind its products of V
  // (sixteen sequences of wide heads 35.0 -> 32.6 us a pass, 1000 positions after 16001 197.5 -> 192). With two in flight
  // that is late already (131000 positions 33.7 -> 34.4).
  constexpr bool EARLY = PF == 1;
  __shared__ __align__(16) float Os[kWaves][16][D + 4];
  __shared__ float2 Ms[kWaves][16];
  const Kv8Dev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col16 = lane & 15, G = lane >> 4;
  // the tiles that read the same blocks run on the same XCD (workgroups go round them in turn), where there are enough
  // units for all of them; fewer than 8 take turns, and none stands for a unit that is not there
  const int id = blockIdx.x, units = a.n_seqs * c.kvh * a.splits;
  const int unit = units < 8 ? id % units : id / 8 / a.tiles * 8 + id % 8;
  const int tile = units < 8 ? id / units : id / 8 % a.tiles;
  if (unit >= units) return;
  const int split = unit % a.splits, hs = unit / a.splits, h = hs % c.kvh, sc = hs / c.kvh, s = a.seq0 + sc;
  const size_t head = (size_t)s * c.kvh + h;
  const int b0 = split * kWaves + w, step = a.splits * kWaves;  // this wave's first block, and on to the next
  const int* table = c.table + head * c.slots;
  int raw = table[min(b0 + lane * step, c.slots - 1)];  // lane x: the slot of this wave's x-th block
  const int len = kv_len(c, s), cols = a.n * a.g;
  const int seen = blocks_seen(len, a.n, a.g, tile, W), used = splits_used(seen, a.splits);
  if (split >= used) return;
  const size_t col0 = (size_t)hs * cols;  // of the workspace's columns

  // The wave's blocks, 64 at a time, lane x holding the x-th one's slot and scales. The first are asked for before the
  // queries are looked at.
  const int full = min(seen, len / kKvBlock);  // blocks that are coded
  int slot_l = 0, count = 0;
  float ks_l = 0.0f, vs_l = 0.0f, lvs_l = 0.0f, ivs_l = 0.0f;
  uint4 kb[PF][2 * CH], vb[PF][2 * CH];
  auto batch = [&](int base) {  // scales() follows, behind the loads of the first blocks
    if (base != b0) raw = table[min(base + lane * step, c.slots - 1)];
    slot_l = kv_slot(c, raw);
    const size_t sl = head * c.slots + slot_l;
    vs_l = gmem(c.vs)[sl];
    ks_l = gmem(c.ks)[sl];
    count = min(64, (full - base + step - 1) / step);
  };
  auto scales = [&]() {
    // a V that is not finite makes the scores NaN, not the scale: columns that see none of the block are masked there
    if (vs_l != vs_l) ks_l = vs_l, vs_l = 1.0f;
    ks_l *= a.kf;
    lvs_l = __builtin_amdgcn_logf(vs_l);
    ivs_l = 1.0f / vs_l;
  };
  auto fetch_k = [&](int p, int x) {
    const int slot = __builtin_amdgcn_readlane(slot_l, min(x, count - 1));
    const size_t at = (head * c.slots + slot) * (size_t)(kKvBlock * D);
    const uint8_t* kp = c.kc + at + col16 * D + G * 16;
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
      for (int z = 0; z < CH; z++)
        kb[p][y * CH + z] = STREAM ? gload_u4_nt(kp + y * 16 * D + z * 64) : gload_u4(kp + y * 16 * D + z * 64);
  };
  auto fetch_v = [&](int p, int x) {
    const int slot = __builtin_amdgcn_readlane(slot_l, min(x, count - 1));
    const size_t at = (head * c.slots + slot) * (size_t)(kKvBlock * D);
    const uint8_t* vp = c.vc + at + (col16 % RP * 4 + G) * (U * 8) + col16 / RP * 16;
#pragma unroll
    for (int y = 0; y < 2 * CH; y++) vb[p][y] = STREAM ? gload_u4_nt(vp + y * 1024) : gload_u4(vp + y * 1024);
  };
  auto fetch = [&](int p, int x) {
    fetch_k(p, x);
    fetch_v(p, x);
  };
  if (b0 < full) {
    batch(b0);
#pragma unroll
    for (int p = 0; p < PF; p++) fetch(p, p);
    __builtin_amdgcn_sched_barrier(0);
  }

  // queries and the rows that each column sees
  h8 qh[NT][KS], ql[NT][F16 ? 1 : KS];
  int qe[NT];  // log2 of what is still to be multiplied by: ke, and what queries of f32 were divided by
  int sees[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int col = tile * W + t * 16 + col16, cc = min(col, cols - 1), i = cc / a.g;
    sees[t] = len - a.n + 1 + i;
    const long long at = sc * a.q.seq + i * a.q.pos + (long long)(h * a.g + cc % a.g) * a.q.head;
    float x[KS][8];
#pragma unroll
    for (int k = 0; k < KS; k++) {
      load8<F16>(a.q, at + (k >> 1) * 64 + G * 16 + (k & 1) * 8, a.vec & 1, x[k]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[k][j] = __uint_as_float(__float_as_uint(x[k][j]) ^ a.sign);
        if constexpr (F16) x[k][j] += x[k][j] - x[k][j];  // inf to NaN, as the difference of f32's halves makes it
      }
    }
    qe[t] = a.ke;
    if constexpr (!F16) {
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) m = __builtin_fmaxf(m, __builtin_fabsf(x[k][j]));
      m = max_stage<16>(m);
      m = max_stage<32>(m);
      const int e = m > 0.0f && m < __int_as_float(0x7f800000) ? __builtin_amdgcn_frexp_expf(m) : 0;
      // 2^(10 - e) in two factors: either alone could leave the type
      const int e1 = (10 - e) / 2, e2 = 10 - e - e1;
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 8; j++) x[k][j] = __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(x[k][j], e1), e2);
      qe[t] += e - 10;
    }
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const _Float16 hi = (_Float16)x[k][j];
        qh[t][k][j] = hi;
        if constexpr (!F16) ql[t][k][j] = (_Float16)(x[k][j] - (float)hi);
      }
  }
  const int sees0 = len - a.n + 1 + min(tile * W, cols - 1) / a.g;  // the least of the tile

  // M + L: the maximum less 7, so that the weights below are 2^7 times those to it; M its part of a score, L of a scale
  // of V, which large scores would round away. l: a lane's own sum
  float M[NT], L[NT], l[NT];
  f4 O[NT][U];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    M[t] = kNone;
    L[t] = l[t] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) O[t][u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  bool far = false;    // some column's M is, or has been, beyond 2^16
  float limit = kShift + kSlack;  // how far beyond M + L a contribution moves it
  float vref = kNone;  // the largest log2 of a scale of V that came with a move of M
  float none = -__builtin_inff();  // opaque, so that eight maxima with it are four instructions
  asm("" : "+s"(none));
  // One block: kop(half, k), vop(u) give the operands, then() runs behind the scores; ks is the scale of K with that of
  // the scores in it, lvs and ivs log2 and inverse of the scale of V. masked: 0, or 1 where some column does not see all
  // of it (S is -inf there, which moves no maximum; NaN with a scale of 0, which moves none either), or 2 for the tail,
  // whose poisoned rows `bad` names.
  auto block = [&](auto masked, auto kop, auto vop, auto then, float ks, float lvs, float ivs, int b, uint32_t bad) {
    constexpr bool MASKED = decltype(masked)::value != 0, TAIL = decltype(masked)::value == 2;
    f4 S[NT][2];
    if constexpr (NT > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < 2; x++) {
#pragma unroll
      for (int t = 0; t < NT; t++) S[t][x] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const h8 ka = kop(x, k);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          S[t][x] = mfma(ka, qh[t][k], S[t][x]);
          if constexpr (!F16) S[t][x] = mfma(ka, ql[t][k], S[t][x]);
        }
      }
    }
    if constexpr (MASKED) {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = x * 16 + G * 4 + i;
            if (bad >> row & 1) S[t][x][i] = __int_as_float(0x7fc00000);
            if (b * kKvBlock + row >= sees[t]) S[t][x][i] = -__builtin_inff();
          }
    }
    if constexpr (NT > 1) __builtin_amdgcn_s_setprio(0);
    then();
    float f[NT], mx[NT], d[NT];
    bool move = false;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      // the three scales of a score meet here, with their exponents in one: no two of them leave f32 where all three
      // do not. The tail has no scale of K that says how small it is: its scores come in 2^24 times.
      if constexpr (TAIL) {
#pragma unroll
        for (int x = 0; x < 8; x++) S[t][x >> 2][x & 3] *= 0x1p24f;
      }
      f[t] = __builtin_amdgcn_ldexpf(ks, TAIL ? qe[t] - 24 : qe[t]);
      mx[t] = none;
#pragma unroll
      for (int x = 0; x < 8; x++) mx[t] = __builtin_fmaxf(mx[t], S[t][x >> 2][x & 3]);
      d[t] = lvs - L[t];
      move |= __builtin_fmaf(mx[t], f[t], d[t] - M[t]) > limit;
    }
    if (__any(move)) {
      vref = __builtin_fmaxf(vref, lvs);
      float y[NT];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        y[t] = max_stage<32>(max_stage<16>(mx[t])) * f[t];
        far |= __any(__builtin_fabsf(y[t]) > 65536.0f && y[t] > kNone);
      }
      if (far) limit = none;  // -inf: from here on every block comes here, and M follows the scores alone
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float yl = far ? kFarL : lvs - kShift;
        const bool up = (y[t] - M[t]) + (yl - L[t]) > 0.0f;
        const float mn = up ? y[t] : M[t], ln = up ? yl : L[t];
        const float al = __builtin_amdgcn_exp2f((M[t] - mn) + (L[t] - ln));
        M[t] = mn;
        L[t] = ln;
        d[t] = lvs - ln;
        l[t] *= al;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) O[t][u][i] *= al;
      }
    }
    const bool apart = far || lvs < vref - kApart;  // the same for the wave
    float k2[NT];                            // p is 2^k2 times what M makes it, and O with it
#pragma unroll
    for (int t = 0; t < NT; t++) k2[t] = 0.0f;
    if (apart) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float y = max_stage<32>(max_stage<16>(mx[t])) * f[t];
        k2[t] = __builtin_floorf((M[t] - y) - (d[t] - kShift));
        k2[t] = __builtin_fminf(__builtin_fmaxf(k2[t], 0.0f), kMostUp);  // of NaN 0
        d[t] += k2[t];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) O[t][u][i] = __builtin_amdgcn_ldexpf(O[t][u][i], (int)k2[t]);
      }
    }
    float c0[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) c0[t] = d[t] - M[t];
    if (far) {  // M is rounded by more than p allows: the same rounding for the scores, and their difference first
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int x = 0; x < 8; x++) S[t][x >> 2][x & 3] = S[t][x >> 2][x & 3] * f[t] - M[t];
        f[t] = 1.0f;
        c0[t] = d[t];
      }
    }
    h8 ph[NT], pl[LO ? NT : 1];
    float part[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float p[8];
#pragma unroll
      for (int x = 0; x < 8; x++) p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][x >> 2][x & 3], f[t], c0[t]));
      if constexpr (MASKED) {
#pragma unroll
        for (int x = 0; x < 8; x++)
          if (b * kKvBlock + (x >> 2) * 16 + G * 4 + (x & 3) >= sees[t]) p[x] = 0.0f;
      }
      part[t] = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
      for (int x = 0; x < 8; x++) {
        ph[t][x] = (_Float16)p[x];
        if constexpr (LO) pl[t][x] = (_Float16)(p[x] - (float)ph[t][x]);
      }
    }
    if constexpr (NT > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const h8 va = vop(u);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        O[t][u] = mfma(va, ph[t], O[t][u]);
        if constexpr (LO) O[t][u] = mfma(va, pl[t], O[t][u]);
      }
    }
    if constexpr (NT > 1) __builtin_amdgcn_s_setprio(0);
    if (apart) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
        part[t] = __builtin_amdgcn_ldexpf(part[t], -(int)k2[t]);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) O[t][u][i] = __builtin_amdgcn_ldexpf(O[t][u][i], -(int)k2[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) l[t] = __builtin_fmaf(part[t], ivs, l[t]);
    if constexpr (TRACK) {  // lanes of group 0 write tile 0's, those of group 2 tile 1's
      static_assert(NT <= 2, "");
      const float y = add16(add32(part[0], part[NT - 1]));
      const float m = G >= 2 ? M[NT - 1] : M[0], ml = G >= 2 ? L[NT - 1] : L[0];
      const int col = tile * W + (G >> 1) * 16 + col16;
      if ((NT == 2 ? !(G & 1) : G == 0) && col < cols)
        a.lse[((size_t)hs * c.slots + b) * cols + col] = __builtin_amdgcn_logf(y) + (ml - lvs) + m;
    }
  };

  for (int base = b0; base < full; base += 64 * step) {
    if (base != b0) {
      batch(base);
#pragma unroll
      for (int p = 0; p < PF; p++) fetch(p, p);
    }
    scales();
    auto run = [&](auto masked, int p, int x, auto then) {
      auto kop = [&](int y, int k) {
        const uint4 v = kb[p][y * CH + (k >> 1)];
        return k & 1 ? half_codes(v.z, v.w) : half_codes(v.x, v.y);
      };
      auto vop = [&](int u) {
        const uint4 v = vb[p][u >> 1];
        return u & 1 ? half_codes(v.z, v.w) : half_codes(v.x, v.y);
      };
      block(masked, kop, vop, then, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_l), x)),
            __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs_l), x)),
            __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ivs_l), x)), base + x * step, 0u);
    };
    // the blocks that every column sees all of, and those that some see a part of
    const int whole = max(0, min(count, (sees0 / kKvBlock - base + step - 1) / step));
    for (int x = 0; x < whole; x += PF) {
#pragma unroll
      for (int p = 0; p < PF; p++) {
        if (x + p < whole) run(std::integral_constant<int, 0>(), p, x + p, [&]() { if constexpr (EARLY) fetch_k(p, x + p + PF); });
        if constexpr (EARLY) fetch_v(p, x + p + PF);
        else fetch(p, x + p + PF);
      }
    }
    for (int x = whole; x < count; x++) {
      if (x) fetch(0, x);
      run(std::integral_constant<int, 1>(), 0, x, []() {});
    }
  }
  if (seen > full && full % step == b0) {  // the tail, in fp16
    const int r = len % kKvBlock;
    const uint32_t bad = c.bad[head], use = ~bad & ((1u << r) - 1u);
    const uint16_t* kt = c.kt + head * kKvBlock * D;
    const uint16_t* vt = c.vt + head * kKvBlock * D;
    auto kop = [&](int y, int k) {
      return *reinterpret_cast<const h8*>(kt + (y * 16 + col16) * D + (k >> 1) * 64 + G * 16 + (k & 1) * 8);
    };
    auto vop = [&](int u) {
      h8 v = *reinterpret_cast<const h8*>(vt + ((elem(u, col16) / U * 4 + G) * U + elem(u, col16) % U) * 8);
#pragma unroll
      for (int j = 0; j < 8; j++)  // what no row has written, or poison, must not meet a weight of 0
        v[j] = use >> (G * 4 + (j & 3) + 16 * (j >> 2)) & 1 ? v[j] : (_Float16)0.0f;
      return v;
    };
    block(std::integral_constant<int, 2>(), kop, vop, []() {}, a.kf, 0.0f, 1.0f, full, bad);
  }

  // the waves' shares, tile by tile
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const float lt = add16(add32(l[t], l[t]));
    if (t) __syncthreads();
    if (G == 0) Ms[w][col16] = make_float2(M[t] + L[t], lt);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int u = 0; u < U; u += 2)
        *reinterpret_cast<float2*>(&Os[w][col16][elem(u, G * 4 + i)]) = make_float2(O[t][u][i], O[t][u + 1][i]);
    __syncthreads();
    const int cl = threadIdx.x >> 4, e0 = (threadIdx.x & 15) * U, col = tile * W + t * 16 + cl;
    if (col < cols) {
      float m = Ms[0][cl].x;
#pragma unroll
      for (int x = 1; x < kWaves; x++) m = __builtin_fmaxf(m, Ms[x][cl].x);
      float sum = 0.0f, o[U] = {};
#pragma unroll
      for (int x = 0; x < kWaves; x++) {
        const float al = __builtin_amdgcn_exp2f(Ms[x][cl].x - m);
        sum = __builtin_fmaf(Ms[x][cl].y, al, sum);
#pragma unroll
        for (int e = 0; e < U; e++) o[e] = __builtin_fmaf(Os[x][cl][e0 + e], al, o[e]);
      }
      const size_t wc = col0 + col;
      if (used == 1) {
        const bool none = sees_none(len, a.n, a.g, col);
        const float inv = none ? 0.0f : 1.0f / sum;
        const long long at = sc * a.out.seq + (long long)(col / a.g) * a.out.pos +
                             (long long)(h * a.g + col % a.g) * a.out.head + e0;
#pragma unroll
        for (int e = 0; e < U; e++) o[e] = F16 ? in_f16(o[e] * inv) : o[e] * inv;
        store_out<U, F16>(a.out, at, a.vec & 2, o);
        if (TRACK && e0 == 0) a.tot[wc] = total_of(m, sum, none);
      } else {
        float* po = a.part + (wc * a.splits + split) * D + e0;
#pragma unroll
        for (int e = 0; e < U; e += 4) *reinterpret_cast<f4*>(po + e) = f4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        if (e0 == 0) a.ml[wc * a.splits + split] = make_float2(m, sum);
      }
    }
  }
}

// A column's maximum and sum over its splits, lane x holding split x's, and the factor of split x's products.
__device__ __forceinline__ void column_sum(const AttnArgs& a, long long wc, int used, int lane, float* m, float* al,
                                           float* sum) {
  const float2 x = a.ml[wc * a.splits + min(lane, a.splits - 1)];
  const bool in = lane < used;
  *m = group_max(in ? x.x : kNone);
  *al = in ? __builtin_amdgcn_exp2f(x.x - *m) : 0.0f;
  *sum = group_sum(in ? x.y * *al : 0.0f);
}

// The splits' shares of a column: C waves to a column, 4 / C columns to a workgroup. The waves take every C-th split's
// products, all of them asked for at once and before the factors are known: the splits that a short sequence leaves
// unused lie in the workspace too, and are not looked at. Bound by latency: 2.7 us behind a short attention (3.4 with
// four loads at a time behind the factors), 4.9 behind one of 134 MB, as any launch there.
template <int D, bool F16, bool TRACK, int C>
__device__ __forceinline__ void combine_column(const AttnArgs& a, int width, int block, float (*Os)[D]) {
  constexpr int E = D / 64, N = C == 4 ? kMaxSplits / 4 : 8;  // a wave's splits, at most
  const Kv8Dev& c = a.c;
  const int cols = a.n * a.g, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long wc = (long long)block * (4 / C) + w / C;
  if (wc >= (long long)a.n_seqs * c.kvh * cols) return;  // C = 4: no column is left out
  const int col = (int)(wc % cols), hs = (int)(wc / cols), h = hs % c.kvh, sc = hs / c.kvh;
  const float* po = a.part + wc * a.splits * D + lane;
  float y[N][E];
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int e = 0; e < E; e++)
      if (w % C + j * C < a.splits) y[j][e] = gmem(po)[(size_t)(w % C + j * C) * D + e * 64];
  const int len = kv_len(c, a.seq0 + sc), used = splits_used(blocks_seen(len, a.n, a.g, col / width, width), a.splits);
  float m, al, sum;
  column_sum(a, wc, used, lane, &m, &al, &sum);
  if (used == 1) return;
  float o[E] = {};
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int split = w % C + j * C;
    if (split < used) {
      const float aj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(al), split));
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(y[j][e], aj, o[e]);
    }
  }
  if constexpr (C == 4) {
#pragma unroll
    for (int e = 0; e < E; e++) Os[w][e * 64 + lane] = o[e];
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int e = 0; e < E; e++)
      o[e] = (o[e] + Os[1][e * 64 + lane]) + (Os[2][e * 64 + lane] + Os[3][e * 64 + lane]);
  }
  const bool none = sees_none(len, a.n, a.g, col);
  const float inv = none ? 0.0f : 1.0f / sum;
  const long long at = sc * a.out.seq + (long long)(col / a.g) * a.out.pos +
                       (long long)(h * a.g + col % a.g) * a.out.head + lane;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if constexpr (F16) ((uint16_t*)a.out.p)[at + e * 64] = f2h(in_f16(o[e] * inv));
    else ((float*)a.out.p)[at + e * 64] = o[e] * inv;
  }
  if (TRACK && lane == 0) a.tot[wc] = total_of(m, sum, none);
}

template <int D, bool F16, bool TRACK, int C>
__global__ __launch_bounds__(256) void k_kv8_combine(AttnArgs a, int width) {
  __shared__ float Os[4][D];
  combine_column<D, F16, TRACK, C>(a, width, blockIdx.x, Os);
}

// A block's weight for a column, at most 1 however far scores beyond 2^16 have rounded the two logarithms; NaN stays.
__device__ __forceinline__ float weight_of(float x) { return __builtin_amdgcn_exp2f(x > 0.0f ? 0.0f : x); }

// mass = decay * mass + the block's weights: P lanes to a block, each with every P-th column, joined pairwise.
__device__ __forceinline__ void mass_block(const AttnArgs& a, int hs, int b, int x, int P, float decay,
                                           const float* tot) {
  const Kv8Dev& c = a.c;
  const int h = hs % c.kvh, s = a.seq0 + hs / c.kvh, len = kv_len(c, s), cols = a.n * a.g;
  if (b * kKvBlock >= len) return;  // all P lanes
  const size_t head = (size_t)s * c.kvh + h;
  const int i0 = max(0, b * kKvBlock - (len - a.n));  // the first position that sees any of the block
  const float* lse = a.lse + ((size_t)hs * c.slots + b) * cols;
  float w = 0.0f;
  for (int col = i0 * a.g + x; col < cols; col += 4 * P) {  // four loads in flight; past the last column its own, for 0
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int at = min(col + j * P, cols - 1);
      y[j] = lse[at] - tot[at];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) w += col + j * P < cols ? weight_of(y[j]) : 0.0f;
  }
  for (int m = P / 2; m; m >>= 1) w += __shfl_xor(w, m);
  if (x) return;
  float* m = c.mass + head * c.slots + kv_slot(c, c.table[head * c.slots + b]);
  *m = __builtin_fmaf(decay, *m, w);
}

__global__ __launch_bounds__(256) void k_kv8_mass(AttnArgs a, float decay, int P) {
  const int hs = blockIdx.z * a.c.kvh + blockIdx.y;
  mass_block(a, hs, blockIdx.x * (256 / P) + threadIdx.x / P, threadIdx.x % P, P, decay,
             a.tot + (size_t)hs * a.n * a.g);
}

// Combine and masses of one tile of columns in one launch: the first workgroups combine, the others, per KV head, form
// the columns' sums from the splits' again instead of waiting for them.
template <int D, bool F16, int C>
__global__ __launch_bounds__(256) void k_kv8_finish(AttnArgs a, int width, int combines, int per_head, float decay,
                                                    int P) {  // per_head: workgroups for the masses of a head
  __shared__ float Os[4][D], tot[16];
  if ((int)blockIdx.x < combines) {
    combine_column<D, F16, false, C>(a, width, blockIdx.x, Os);
    return;
  }
  const int x = blockIdx.x - combines, hs = x / per_head, lane = threadIdx.x & 63, cols = a.n * a.g;
  // lane `col` of a block's P holds its column; all that does not wait for the sums is asked for first
  const Kv8Dev& c = a.c;
  const int h = hs % c.kvh, s = a.seq0 + hs / c.kvh, col = threadIdx.x % P;
  const int b = min(x % per_head * (256 / P) + (int)threadIdx.x / P, c.slots - 1);
  const size_t head = (size_t)s * c.kvh + h;
  const float lse = gmem(a.lse)[((size_t)hs * c.slots + b) * cols + min(col, cols - 1)];
  float* mass = c.mass + head * c.slots + kv_slot(c, gmem(c.table)[head * c.slots + b]);
  const float old = gmem(mass)[0];
  const int len = kv_len(c, s), used = splits_used(blocks_seen(len, a.n, a.g, 0, width), a.splits);
  for (int i = threadIdx.x >> 6; i < cols; i += 4) {
    float m, al, sum;
    column_sum(a, (long long)hs * cols + i, used, lane, &m, &al, &sum);
    if (lane == 0)
      tot[i] = used == 1 ? a.tot[(size_t)hs * cols + i] : total_of(m, sum, sees_none(len, a.n, a.g, i));
  }
  __syncthreads();
  // a column's position sees some of the block, and the block is the last thread group's own (the index is clamped)
  const bool mine = x % per_head * (256 / P) + (int)threadIdx.x / P == b && b * kKvBlock < len;
  float w = col < cols && b * kKvBlock < len - a.n + 1 + col / a.g ? weight_of(lse - tot[col]) : 0.0f;
  for (int m = P / 2; m; m >>= 1) w += __shfl_xor(w, m);
  if (mine && col == 0) *mass = __builtin_fmaf(decay, old, w);
}

int tile_count(int cols) { return cols <= 16 ? 1 : 2; }  // tiles of 16 columns of a wave

}  // namespace

KvAttnPlan kv8_attn_plan(const Kv8Dev& c, int n_seqs, int heads, int n, bool track) {
  KvAttnPlan p;
  const int cols1 = heads / c.kvh * n, nt = tile_count(cols1), tiles = (cols1 + 16 * nt - 1) / (16 * nt);
  const size_t cols = (size_t)n_seqs * heads * n;
  const long long units = (long long)n_seqs * c.kvh * tiles;
  // Splits cost a second launch and the partials' way through memory: one workgroup for each of 256 compute units, and
  // more (up to 1024, four to a unit) only while a wave keeps 16 blocks of a full cache; never fewer than 3 a wave. With
  // 1024 workgroups wherever they could be had, a pass over sixteen sequences of wide heads takes 39 us for 32.6, 300
  // positions after 1000 in f32 39.7 for 30.8; with 256 at most, eight sequences of up to 100003 take 162 for 125, though
  // 200 positions after 4000 of wide heads 54 for 64.
  const int cap = c.slots / (kWaves * 3), most = cap < 1 ? 1 : cap > kMaxSplits ? kMaxSplits : cap;
  long long s = 256 / units > 1 ? 256 / units : 1;
  while (2 * s * units <= 1024 && c.slots / (2 * s * kWaves) >= 16) s *= 2;
  p.splits = (int)(s < most ? s : most);
  // Sizes that grow with every argument, so that a workspace does for all smaller calls: splits * units is at most 1024,
  // a unit at most 32 columns.
  const size_t shares = most > 1 ? (cols * most < 32768 ? cols * most : 32768) : 0;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p.tot = 0;
  p.ml = up(cols * 4);
  p.parts = p.ml + up(shares * 8);
  p.lse = p.parts + up(shares * c.d * 4);
  p.bytes = p.lse + (track ? cols * c.slots * 4 : 0);
  return p;
}

namespace {

template <int D, bool F16, bool TRACK>
hipError_t attend(hipStream_t s, AttnArgs a, float decay) {
  const int cols = a.n * a.g, nt = tile_count(cols), width = 16 * nt;
  a.tiles = (cols + width - 1) / width;
  const long long units = (long long)a.n_seqs * a.c.kvh * a.splits;
  const long long grid = (units < 8 ? units : (units + 7) / 8 * 8) * a.tiles;  // below 2^23 (256 threads each: 2^31)
  // A layer's cache of 96 MB and more is streamed past the others: three of them outgrow the 256 MB last-level cache, and
  // a model has more. 565 MB of eight sequences 138 -> 125 us a pass, 134 MB of one 35.7 -> 33.7; where three caches
  // still fit (68 MB in use of 134 each), a pass loses what it would find there, 31.5 -> 32.6.
  const bool stream = nt == 1 && 2ll * a.n_seqs * a.c.kvh * a.c.max_len * D >= 96ll << 20;
  if (stream) klaunch(k_kv8_attend<D, F16, 1, TRACK, true>, (unsigned)grid, kWaves * 64, 0, s, a);
  else if (nt == 1) klaunch(k_kv8_attend<D, F16, 1, TRACK, false>, (unsigned)grid, kWaves * 64, 0, s, a);
  else klaunch(k_kv8_attend<D, F16, 2, TRACK, false>, (unsigned)grid, kWaves * 64, 0, s, a);
  // what follows reads the workspace that this launch writes, and the masses are the caller's
  if (const hipError_t e = hipGetLastError()) return e;
  const long long all = (long long)a.n_seqs * a.c.kvh * cols;
  int P = 1;
  while (P < cols && P < 64) P *= 2;
  const int per_head = (a.c.slots * P + 255) / 256;
  if (TRACK && a.splits > 1 && cols <= 16) {
    // splits mean fewer than 1024 heads: the grid stays small. (A fifth as many workgroups, each with more blocks of a
    // head, took 11.6 us for 9.2: the blocks' loads wait for each other.)
    const int C = a.splits > 8 ? 4 : 1, combines = (int)((all * C + 3) / 4);
    const unsigned both = (unsigned)(combines + all / cols * per_head);
    if (C == 4) klaunch(k_kv8_finish<D, F16, 4>, both, 256, 0, s, a, width, combines, per_head, decay, P);
    else klaunch(k_kv8_finish<D, F16, 1>, both, 256, 0, s, a, width, combines, per_head, decay, P);
    return hipGetLastError();
  }
  if (a.splits > 8) klaunch(k_kv8_combine<D, F16, TRACK, 4>, (unsigned)all, 256, 0, s, a, width);
  else if (a.splits > 1) klaunch(k_kv8_combine<D, F16, TRACK, 1>, (unsigned)((all + 3) / 4), 256, 0, s, a, width);
  if (const hipError_t e = hipGetLastError()) return e;
  if (TRACK) klaunch(k_kv8_mass, dim3(per_head, a.c.kvh, a.n_seqs), 256, 0, s, a, decay, P);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_attend(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int heads, int n, float scale,
                             KvRows q, KvRows out, float decay, void* ws) {
  const bool track = decay >= 0.0f;
  int ke;
  const float kf = frexpf(__builtin_fabsf(scale), &ke) * kLog2e;
  const KvAttnPlan p = kv8_attn_plan(c, n_seqs, heads, n, track);
  char* w = (char*)ws;
  AttnArgs a{c, q, out, seq0, n_seqs, heads / c.kvh, n, p.splits, 1, wide_rows(q) | wide_rows(out) << 1,
             kf, ke, scale < 0.0f ? 0x80000000u : 0u, (float*)(w + p.parts), (float2*)(w + p.ml), (float*)(w + p.tot),
             track ? (float*)(w + p.lse) : nullptr};
#define ATT(DD, FF) \
  if (c.d == DD && q.f16 == FF) return track ? attend<DD, FF, true>(s, a, decay) : attend<DD, FF, false>(s, a, decay);
  ATT(64, 0) ATT(64, 1) ATT(128, 0) ATT(128, 1)
#undef ATT
  return hipErrorInvalidValue;
}

}  // namespace moert
