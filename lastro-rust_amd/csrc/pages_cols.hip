// Attention of few rows over the paged 16-bit K/V cache (pages.h), on the matrix cores with f32 sums; and the join of
// splits.
//
// A row is one query head at one position; the rows of a KV head's group, position by position, go in tiles of 16. The
// waves of a workgroup take the blocks of 32 positions in turn, each for itself, and join in LDS;
// where tiles are too few for the device several workgroups share one (splits) and a second launch joins them. Per block:
//   S = K Q^T    MFMA 16x16x32, rows = positions, columns = rows of the tile. Row i of product x is position
//                16 (i / 8) + 8 x + i % 8, so that a lane of group G = lane / 16 gets the 8 positions that lie side by
//                side in V: 16 (G / 2) + 4 (G % 2) + 0 .. 3, and 8 on.
//   softmax      p = 2^(S f - M), f = scale log2 e; M, the running maximum less 7, moves only for weights above 2^15 (or, where
//                scores are far from 0, above 2^7).
//   O += V^T P^T MFMA 16x16x32, rows = elements; p, as two numbers of the cache's type, never leaves its lane.
// A wave's blocks go to its own ring in LDS, one being worked on while the next is on its way; nobody waits for another
// wave. (Straight into registers, where the compiler kept one in flight, 131000 positions of 8 KV heads of 64 took 87 us for
// 39.)
//
// What bounds it, measured on one MI355X: the cache's bytes. 973 MB of 43 sequences (8 KV heads of 128, bf16) in 146 us, 6.6
// TB/s (a copy of 1 GiB reaches 5.2, reading and writing); 268 MB of one in 39, part of it from the last-level cache. Short
// caches: launches and four loads that wait for each other (4.6 us for 100 rows). Reads of K take two turns in LDS for one
// (rows 8 apart share banks), a third of its cycles, which nothing waits for.
#include <type_traits>

#include "pages_dev.h"

namespace moert {

namespace {

constexpr int kWaves = 4;

__device__ __forceinline__ float sum16(float x) {
  x += partner<16>(x);
  return x + partner<32>(x);
}

// Blocks that a tile's last row sees; splits of it that have any.
__device__ __forceinline__ int tile_blocks(const PgArgs& a, const PgTile& t, int w) {
  return (max(0, t.sees0 + (min(t.row0 + w, t.rows) - 1) / a.g) + kPgBlock - 1) / kPgBlock;
}
__device__ __forceinline__ int cols_used(const PgArgs& a, int blocks) {
  return max(1, min(a.splits, (blocks + kWaves - 1) / kWaves));
}

template <int D, int T, bool STREAM>
__global__ __launch_bounds__(kWaves * 64, D == 64 ? 2 : 1) void k_pages_cols(PgArgs a) {
  constexpr int KS = D / 32, U = D / 16, RING = 2;             // blocks in flight, and being worked on
  constexpr int kBytes = 64 * D, kCopies = 2 * kBytes / 1024;  // of a block of K or V; of both
  constexpr bool LO = T == PG_F32;                                                     // queries as two fp16
  __shared__ __align__(16) uint8_t ring[kWaves][RING][2][kBytes];
  __shared__ float2 Ms[kWaves][16];
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, G = lane >> 4;
  const int id = blockIdx.x, h = id % c.kvh, split = id / c.kvh % a.splits, y = id / c.kvh / a.splits;
  PgTile t;
  if (!pg_tile(a, y, 16, &t)) return;
  const int blocks = tile_blocks(a, t, 16), used = cols_used(a, blocks);
  if (split >= used) return;
  // this wave's blocks: b0, b0 + step, ..; lane x holds the place in the pool of the x-th of 64
  const int b0 = split * kWaves + w, step = a.splits * kWaves, count = max(0, (blocks - b0 + step - 1) / step);
  const int* table = c.table + (size_t)t.s * c.max_pages;
  const uint32_t into = pg_lds(ring[w]);
  int place = 0;
  auto fetch = [&](int x) {
    if (x % 64 == 0) {
      const int b = min(b0 + (x + lane) * step, blocks - 1);
      place = pg_block(c, pg_page(c, gmem(table)[b >> (c.lp - 5)]), h, b);
    }
    const size_t at = (size_t)__builtin_amdgcn_readlane(place, x % 64) * kBytes;
    const uint32_t to = into + x % RING * (2 * kBytes);
    pg_copy_to_lds<kCopies / 2, STREAM>((const uint8_t*)c.k + at, lane * 16, to);
    pg_copy_to_lds<kCopies / 2, STREAM>((const uint8_t*)c.v + at, lane * 16, to + kBytes);
  };
#pragma unroll
  for (int x = 0; x < RING; x++)
    if (x < count) fetch(x);

  // queries, and the rows that each column sees
  const int row = min(t.row0 + col, t.rows - 1), i = row / a.g;
  const int sees = t.sees0 + i, least = t.sees0 + t.row0 / a.g, len = t.sees0 + t.rows / a.g - 1;
  uint4 qh[KS], ql[LO ? KS : 1];
  int qe = 0;
  {
    const long long at = (long long)(t.lo + i) * a.q.pos + (long long)(h * a.g + row % a.g) * a.q.head + G * 8;
    if constexpr (LO) {
      float v[KS][8], m = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        pg_query<T>(a, at + k * 32, v[k]);
#pragma unroll
        for (int j = 0; j < 8; j++) m = __builtin_fmaxf(m, __builtin_fabsf(v[k][j]));
      }
      m = max_stage<32>(max_stage<16>(m));
      qe = pg_split_exp(m);
#pragma unroll
      for (int k = 0; k < KS; k++) pg_split<T>(v[k], qe, &qh[k], &ql[k]);
    } else {
#pragma unroll
      for (int k = 0; k < KS; k++) qh[k] = pg_query16<T>(a, at + k * 32);
    }
  }
  const float f = pg_factor(a, qe);

  float Sm = kPgNone, M = kPgNone, l = 0.0f;  // the maximum as a sum of products, and times f; a lane's own sum
  pg_f4 O[U];
#pragma unroll
  for (int u = 0; u < U; u++) O[u] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
  bool far = false;
  float none = -__builtin_inff();
  asm("" : "+s"(none));

  auto block = [&](auto masked, const uint8_t* kp, const uint8_t* vp, int b) {
    constexpr bool MASKED = decltype(masked)::value;
    pg_f4 S[2];
#pragma unroll
    for (int z = 0; z < 2; z++) {
      S[z] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const uint4 ka = *reinterpret_cast<const uint4*>(kp + ((4 * k + G) * kPgBlock + col / 8 * 16 + col % 8 + 8 * z) * 16);
        S[z] = pg_mfma<T>(ka, qh[k], S[z]);
        if constexpr (LO) S[z] = pg_mfma<T>(ka, ql[k], S[z]);
      }
    }
    const int t0 = b * kPgBlock + G / 2 * 16 + G % 2 * 4;  // the lane's first position
    if constexpr (MASKED) {
#pragma unroll
      for (int z = 0; z < 8; z++)
        if (t0 + z / 4 * 8 + z % 4 >= sees) S[z / 4][z % 4] = -__builtin_inff();
    }
    float mx = none;
#pragma unroll
    for (int z = 0; z < 8; z++) mx = __builtin_fmaxf(mx, S[z / 4][z % 4]);
    // Far from 0 the maximum moves for any score above it: there M is rounded by more than the slack leaves.
    if (__any(far ? mx > Sm : __builtin_fmaf(mx, f, -M) > kPgSlack)) {
      const float m = __builtin_fmaxf(Sm, max_stage<32>(max_stage<16>(mx)));
      const float to = __builtin_fmaxf(__builtin_fmaf(m, f, -kPgShift), kPgNone);  // finite where nothing is seen yet
      far |= __any(__builtin_fabsf(to) > kPgFar && m > kPgNone);
      const float al = __builtin_amdgcn_exp2f(far ? (Sm - m) * f : M - to);  // as the weights were taken
      Sm = m;
      M = to;
      l *= al;
#pragma unroll
      for (int u = 0; u < U; u++) O[u] *= al;
    }
    float x[8];
    if (far) {
#pragma unroll
      for (int z = 0; z < 8; z++) x[z] = __builtin_fmaf(S[z / 4][z % 4] - Sm, f, kPgShift);
    } else {
#pragma unroll
      for (int z = 0; z < 8; z++) x[z] = __builtin_fmaf(S[z / 4][z % 4], f, -M);
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float pa = __builtin_amdgcn_exp2f(x[2 * j]), pb = __builtin_amdgcn_exp2f(x[2 * j + 1]);
      l += pa;
      l += pb;
      hi[j] = pg_pack<T>(pa, pb);
      lo[j] = pg_rest<T>(hi[j], pa, pb);
    }
    const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]), pl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    uint32_t keep[4];  // memory behind the sequence's rows may hold anything, and 0 times that would be NaN
    if constexpr (MASKED) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int at = t0 + j / 2 * 8 + j % 2 * 2;
        keep[j] = (at < len ? 0xffffu : 0u) | (at + 1 < len ? 0xffff0000u : 0u);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      uint4 va = *reinterpret_cast<const uint4*>(vp + (G * D + 16 * u + col) * 16);
      if constexpr (MASKED) va = make_uint4(va.x & keep[0], va.y & keep[1], va.z & keep[2], va.w & keep[3]);
      O[u] = pg_mfma<T>(va, ph, O[u]);
      O[u] = pg_mfma<T>(va, pl, O[u]);
    }
  };

  for (int x = 0; x < count; x++) {
    if (x + RING <= count) pg_wait_copies<(RING - 1) * kCopies>();
    else pg_wait_copies<0>();
    const int b = b0 + x * step;
    const uint8_t *kp = ring[w][x % RING][0], *vp = ring[w][x % RING][1];
    if ((b + 1) * kPgBlock > least) block(std::true_type{}, kp, vp, b);
    else block(std::false_type{}, kp, vp, b);
    if (x + RING < count) {
      pg_wait_reads();
      fetch(x + RING);
    }
  }

  // the waves' shares; a wave without blocks has none
  l = sum16(l);
  auto shares = [&](int x) { return reinterpret_cast<float(*)[D + 4]>(&ring[x]); };  // of a wave, where its blocks were
  static_assert(sizeof(float) * 16 * (D + 4) <= RING * 2 * kBytes, "");
  pg_wait_reads();
#pragma unroll
  for (int u = 0; u < U; u++) *reinterpret_cast<pg_f4*>(&shares(w)[col][16 * u + 4 * G]) = O[u];
  if (G == 0) Ms[w][col] = make_float2(M, l);
  __syncthreads();
  const int cl = threadIdx.x / 16, e0 = threadIdx.x % 16 * U, r = t.row0 + cl;
  if (r >= t.rows) return;
  float m = Ms[0][cl].x;
#pragma unroll
  for (int x = 1; x < kWaves; x++) m = __builtin_fmaxf(m, Ms[x][cl].x);
  float sum = 0.0f, o[U] = {};
#pragma unroll
  for (int x = 0; x < kWaves; x++) {
    const float al = __builtin_amdgcn_exp2f(Ms[x][cl].x - m);
    sum = __builtin_fmaf(Ms[x][cl].y, al, sum);
#pragma unroll
    for (int e = 0; e < U; e++) o[e] = __builtin_fmaf(shares(x)[cl][e0 + e], al, o[e]);
  }
  if (used == 1) {
    const float inv = t.sees0 + r / a.g > 0 ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int e = 0; e < U; e++) o[e] *= inv;
    pg_store<T, U>(a, (long long)(t.lo + r / a.g) * a.out.pos + (long long)(h * a.g + r % a.g) * a.out.head + e0, o);
  } else {
    const size_t wc = (((size_t)h * a.tiles + y) * 16 + cl) * a.splits + split;
#pragma unroll
    for (int e = 0; e < U; e += 4)
      *reinterpret_cast<pg_f4*>(a.part + wc * D + e0 + e) = pg_f4{o[e], o[e + 1], o[e + 2], o[e + 3]};
    if (e0 == 0) a.ml[wc] = make_float2(m, sum);
  }
}

// The splits' shares of a row, more than 8 of them: a workgroup to a row, its waves take every fourth split. All products
// are asked for at once and before it is known which splits have any: the others lie in the workspace too, and are not
// looked at.
template <int D, int T, int W>
__global__ __launch_bounds__(256) void k_pages_join(PgArgs a, int rows) {
  constexpr int E = D / 64, N = kPgMaxSplits / 4;
  __shared__ float Os[4][D];
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x, h = id % c.kvh, x = id / c.kvh % rows, y = id / c.kvh / rows;
  const size_t wc = (((size_t)h * a.tiles + y) * W + x) * a.splits;
  const float2 ml = a.ml[wc + min(lane, a.splits - 1)];
  float p[N][E];
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int e = 0; e < E; e++)
      if (w + 4 * j < a.splits) p[j][e] = gmem(a.part)[(wc + w + 4 * j) * D + e * 64 + lane];
  PgTile t;
  if (!pg_tile(a, y, W, &t)) return;
  const int blocks = tile_blocks(a, t, W), used = W == 16 ? cols_used(a, blocks) : pg_tiles_used(a, blocks);
  const int r = t.row0 + x;
  if (used == 1 || r >= t.rows) return;
  const float m = group_max(lane < used ? ml.x : kPgNone);
  const float al = lane < used ? __builtin_amdgcn_exp2f(ml.x - m) : 0.0f;
  const float sum = group_sum(lane < used ? ml.y * al : 0.0f);
  float o[E] = {};
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int s = w + 4 * j;
    if (s < used) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(al), s));
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(p[j][e], f, o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) Os[w][e * 64 + lane] = o[e];
  __syncthreads();
  if (w) return;
  const float inv = t.sees0 + r / a.g > 0 ? 1.0f / sum : 0.0f;
  const long long at = (long long)(t.lo + r / a.g) * a.out.pos + (long long)(h * a.g + r % a.g) * a.out.head + lane;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float v = ((o[e] + Os[1][e * 64 + lane]) + (Os[2][e * 64 + lane] + Os[3][e * 64 + lane])) * inv;
    if constexpr (T == PG_F32) ((float*)a.out.p)[at + e * 64] = v;
    else ((uint16_t*)a.out.p)[at + e * 64] = (uint16_t)pg_pack<T>(pg_clip<T>(v), 0.0f);
  }
}

// The same for up to 8 splits: a lane to four elements of a row, 1024 / D rows to a workgroup.
template <int D, int T, int W>
__global__ __launch_bounds__(256) void k_pages_join_few(PgArgs a, int rows) {
  constexpr int L = D / 4, R = 256 / L, N = 8;
  const PagesDev& c = a.c;
  const int per = (rows + R - 1) / R, id = blockIdx.x, h = id % c.kvh, y = id / c.kvh / per;
  const int x = id / c.kvh % per * R + threadIdx.x / L, e = threadIdx.x % L * 4;
  const size_t wc = (((size_t)h * a.tiles + y) * W + min(x, W - 1)) * a.splits;
  float2 ml[N];
  float4 p[N];
#pragma unroll
  for (int j = 0; j < N; j++)
    if (j < a.splits) {
      ml[j] = a.ml[wc + j];
      p[j] = gload_f4(a.part + (wc + j) * D + e);
    }
  PgTile t;
  if (!pg_tile(a, y, W, &t)) return;
  const int blocks = tile_blocks(a, t, W), used = W == 16 ? cols_used(a, blocks) : pg_tiles_used(a, blocks);
  const int r = t.row0 + x;
  if (used == 1 || x >= rows || r >= t.rows) return;
  float m = ml[0].x;
#pragma unroll
  for (int j = 1; j < N; j++)
    if (j < used) m = __builtin_fmaxf(m, ml[j].x);
  float sum = 0.0f, o[4] = {};
#pragma unroll
  for (int j = 0; j < N; j++)
    if (j < used) {
      const float al = __builtin_amdgcn_exp2f(ml[j].x - m);
      sum = __builtin_fmaf(ml[j].y, al, sum);
      o[0] = __builtin_fmaf(p[j].x, al, o[0]), o[1] = __builtin_fmaf(p[j].y, al, o[1]);
      o[2] = __builtin_fmaf(p[j].z, al, o[2]), o[3] = __builtin_fmaf(p[j].w, al, o[3]);
    }
  const float inv = t.sees0 + r / a.g > 0 ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] *= inv;
  pg_store<T, 4>(a, (long long)(t.lo + r / a.g) * a.out.pos + (long long)(h * a.g + r % a.g) * a.out.head + e, o);
}

}  // namespace

hipError_t launch_pages_cols(hipStream_t s, PgArgs a) {
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * a.splits;
  // Two blocks to a wave: with four narrow ones 42 us for 38.7 (131000 positions of 8 heads of 64), with one wide one 154
  // for 147 (64 sequences, 973 MB). Caches that outgrow the last-level cache in three layers are streamed past it: 174.8 us
  // with one wide block without, 153.8 with the hint; rows whose tiles read the cache again find it there.
  const PagesDev& c = a.c;
  const long long held = (long long)(c.pages < (long long)c.seqs * c.max_pages ? c.pages : (long long)c.seqs * c.max_pages);
  const bool stream = a.most == 1 && a.g <= 16 && ((held * c.kvh * c.d) << c.lp) * 4 >= 96ll << 20;
#define COLS(DD, TT)                                                                              \
  if (c.d == DD && a.q.f16 == TT) {                                                               \
    if (stream) klaunch(k_pages_cols<DD, TT, true>, grid, kWaves * 64, 0, s, a);                  \
    else klaunch(k_pages_cols<DD, TT, false>, grid, kWaves * 64, 0, s, a);                        \
  }
  COLS(64, 0) COLS(64, 1) COLS(64, 2) COLS(128, 0) COLS(128, 1) COLS(128, 2)
#undef COLS
  return hipGetLastError();
}

hipError_t launch_pages_join(hipStream_t s, PgArgs a, int width) {
  const int rows = a.most > 1 || a.g > width ? width : a.g;  // of one position there are no more
  const int per = a.splits > 8 ? rows : (rows * a.c.d / 4 + 255) / 256;
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * per;
#define JOIN(DD, TT, WW)                                                                 \
  if (a.c.d == DD && a.q.f16 == TT && width == WW) {                                     \
    if (a.splits > 8) klaunch(k_pages_join<DD, TT, WW>, grid, 256, 0, s, a, rows);       \
    else klaunch(k_pages_join_few<DD, TT, WW>, grid, 256, 0, s, a, rows);                \
  }
#define JOINS(DD, TT) JOIN(DD, TT, 16) JOIN(DD, TT, 128)
  JOINS(64, 0) JOINS(64, 1) JOINS(64, 2) JOINS(128, 0) JOINS(128, 1) JOINS(128, 2)
#undef JOINS
#undef JOIN
  return hipGetLastError();
}

}  // namespace moert
