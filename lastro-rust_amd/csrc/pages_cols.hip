// Attention of few rows over the paged 16-bit K/V cache (pages.h), on the matrix cores with f32 sums; and the join of
// splits.
//
// A row is one query head at one position; the rows of a KV head's group, position by position, go in tiles of 16. The
// waves of a workgroup take the blocks of 32 positions in turn, straight from memory into registers, and join in LDS;
// where tiles are too few for the device several workgroups share one (splits) and a second launch joins them. Per block:
//   S = K Q^T    MFMA 16x16x32, rows = positions, columns = rows of the tile. Row i of product x is position
//                16 (i / 8) + 8 x + i % 8, so that a lane of group G = lane / 16 gets the 8 positions that lie side by
//                side in V: 16 (G / 2) + 4 (G % 2) + 0 .. 3, and 8 on.
//   softmax      p = 2^(S f - M), f = scale log2 e; the running maximum M moves only for weights above 2^8.
//   O += V^T P^T MFMA 16x16x32, rows = elements; p, as two numbers of the cache's type, never leaves its lane.
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

template <int D, int T>
__global__ __launch_bounds__(kWaves * 64, D == 64 ? 4 : 2) void k_pages_cols(PgArgs a) {
  constexpr int KS = D / 32, U = D / 16, PF = D == 64 ? 2 : 1;  // blocks in flight
  constexpr bool LO = T == PG_F32;                              // queries as two fp16
  __shared__ __align__(16) float Os[kWaves][16][D + 4];
  __shared__ float2 Ms[kWaves][16];
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, G = lane >> 4;
  const int id = blockIdx.x, h = id % c.kvh, split = id / c.kvh % a.splits, y = id / c.kvh / a.splits;
  PgTile t;
  if (!pg_tile(a, y, 16, &t)) return;
  const int blocks = tile_blocks(a, t, 16), used = cols_used(a, blocks);
  if (split >= used) return;
  const int b0 = split * kWaves + w, step = a.splits * kWaves;  // this wave's first block, and on to the next

  // the wave's blocks, 64 at a time, lane x holding the x-th one's place in the pool
  const int* table = c.table + (size_t)t.s * c.max_pages;
  const int lb = c.lp - 5;
  int block_l = 0, count = 0;
  uint4 kb[PF][2 * KS], vb[PF][U];
  auto batch = [&](int base) {
    const int b = min(base + lane * step, blocks - 1);
    block_l = pg_block(c, pg_page(c, gmem(table)[b >> lb]), h, b);
    count = min(64, (blocks - base + step - 1) / step);
  };
  auto fetch_k = [&](int p, int x) {
    const int b = __builtin_amdgcn_readlane(block_l, min(x, count - 1));
    const uint16_t* at = c.k + (size_t)b * (kPgBlock * D) + (G * kPgBlock + col / 8 * 16 + col % 8) * 8;
#pragma unroll
    for (int z = 0; z < 2; z++)
#pragma unroll
      for (int k = 0; k < KS; k++) kb[p][z * KS + k] = gload_u4(at + (k * 4 * kPgBlock + z * 8) * 8);
  };
  auto fetch_v = [&](int p, int x) {
    const int b = __builtin_amdgcn_readlane(block_l, min(x, count - 1));
    const uint16_t* at = c.v + (size_t)b * (kPgBlock * D) + (G * D + col) * 8;
#pragma unroll
    for (int u = 0; u < U; u++) vb[p][u] = gload_u4(at + u * 128);
  };
  if (b0 < blocks) {
    batch(b0);
#pragma unroll
    for (int p = 0; p < PF; p++) {
      fetch_k(p, p);
      fetch_v(p, p);
    }
  }

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

  auto block = [&](auto masked, int p, int b, int next) {
    constexpr bool MASKED = decltype(masked)::value;
    pg_f4 S[2];
#pragma unroll
    for (int z = 0; z < 2; z++) {
      S[z] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        S[z] = pg_mfma<T>(kb[p][z * KS + k], qh[k], S[z]);
        if constexpr (LO) S[z] = pg_mfma<T>(kb[p][z * KS + k], ql[k], S[z]);
      }
    }
    const int t0 = b * kPgBlock + G / 2 * 16 + G % 2 * 4;  // the lane's first position
    if constexpr (MASKED) {
#pragma unroll
      for (int z = 0; z < 8; z++)
        if (t0 + z / 4 * 8 + z % 4 >= sees) S[z / 4][z % 4] = -__builtin_inff();
    }
    if (next < count) fetch_k(p, next);
    float mx = none;
#pragma unroll
    for (int z = 0; z < 8; z++) mx = __builtin_fmaxf(mx, S[z / 4][z % 4]);
    if (__any(__builtin_fmaf(mx, f, -M) > kPgSlack)) {
      const float m = __builtin_fmaxf(Sm, max_stage<32>(max_stage<16>(mx)));
      const float al = __builtin_amdgcn_exp2f((Sm - m) * f);
      Sm = m;
      M = __builtin_fmaxf(m * f, kPgNone);  // finite where nothing is seen yet
      far |= __any(__builtin_fabsf(M) > kPgFar && m > kPgNone);
      l *= al;
#pragma unroll
      for (int u = 0; u < U; u++) O[u] *= al;
    }
    float x[8];
    if (far) {
#pragma unroll
      for (int z = 0; z < 8; z++) x[z] = (S[z / 4][z % 4] - Sm) * f;
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
      const pg_f2 back = pg_unpack<T>(hi[j]);
      lo[j] = pg_pack<T>(pa - back.x, pb - back.y);
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
      uint4 va = vb[p][u];
      if constexpr (MASKED) va = make_uint4(va.x & keep[0], va.y & keep[1], va.z & keep[2], va.w & keep[3]);
      O[u] = pg_mfma<T>(va, ph, O[u]);
      O[u] = pg_mfma<T>(va, pl, O[u]);
    }
    if (next < count) fetch_v(p, next);
  };

  for (int base = b0; base < blocks; base += 64 * step) {
    if (base != b0) {
      batch(base);
#pragma unroll
      for (int p = 0; p < PF; p++) {
        fetch_k(p, p);
        fetch_v(p, p);
      }
    }
    for (int x = 0; x < count; x += PF) {
#pragma unroll
      for (int p = 0; p < PF; p++) {
        const int b = base + (x + p) * step;
        if (PF > 1 && x + p >= count) break;
        if ((b + 1) * kPgBlock > least) block(std::true_type{}, p, b, x + p + PF);
        else block(std::false_type{}, p, b, x + p + PF);
      }
    }
  }

  // the waves' shares; a wave without blocks has none
  l = sum16(l);
#pragma unroll
  for (int u = 0; u < U; u++) *reinterpret_cast<pg_f4*>(&Os[w][col][16 * u + 4 * G]) = O[u];
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
    for (int e = 0; e < U; e++) o[e] = __builtin_fmaf(Os[x][cl][e0 + e], al, o[e]);
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

// The splits' shares of 16 rows of a tile of W, a wave to four of them.
template <int D, int T, int W>
__global__ __launch_bounds__(256) void k_pages_join(PgArgs a) {
  constexpr int E = D / 64, P = W / 16;
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = blockIdx.x, h = id % c.kvh, part = id / c.kvh % P, y = id / c.kvh / P;
  PgTile t;
  if (!pg_tile(a, y, W, &t)) return;
  const int blocks = tile_blocks(a, t, W), used = W == 16 ? cols_used(a, blocks) : pg_tiles_used(a, blocks);
  if (used == 1) return;
  for (int j = 0; j < 4; j++) {
    const int x = part * 16 + w * 4 + j, r = t.row0 + x;
    if (r >= t.rows) return;
    const size_t wc = (((size_t)h * a.tiles + y) * W + x) * a.splits;
    const float2 ml = a.ml[wc + min(lane, used - 1)];
    const float m = group_max(lane < used ? ml.x : kPgNone);
    const float al = lane < used ? __builtin_amdgcn_exp2f(ml.x - m) : 0.0f;
    const float sum = group_sum(lane < used ? ml.y * al : 0.0f);
    float o[E] = {};
#pragma unroll 8
    for (int s = 0; s < used; s++) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(al), s));
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = __builtin_fmaf(gmem(a.part)[(wc + s) * D + lane * E + e], f, o[e]);
    }
    const float inv = t.sees0 + r / a.g > 0 ? 1.0f / sum : 0.0f;
    const long long at = (long long)(t.lo + r / a.g) * a.out.pos + (long long)(h * a.g + r % a.g) * a.out.head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) {
      if constexpr (T == PG_F32) ((float*)a.out.p)[at + e] = o[e] * inv;
      else ((uint16_t*)a.out.p)[at + e] = (uint16_t)pg_pack<T>(pg_clip<T>(o[e] * inv), 0.0f);
    }
  }
}

}  // namespace

hipError_t launch_pages_cols(hipStream_t s, PgArgs a) {
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * a.splits;
#define COLS(DD, TT) \
  if (a.c.d == DD && a.q.f16 == TT) klaunch(k_pages_cols<DD, TT>, grid, kWaves * 64, 0, s, a);
  COLS(64, 0) COLS(64, 1) COLS(64, 2) COLS(128, 0) COLS(128, 1) COLS(128, 2)
#undef COLS
  return hipGetLastError();
}

hipError_t launch_pages_join(hipStream_t s, PgArgs a, int width) {
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * (width / 16);
#define JOIN(DD, TT)                                                                   \
  if (a.c.d == DD && a.q.f16 == TT) {                                                  \
    if (width == 16) klaunch(k_pages_join<DD, TT, 16>, grid, 256, 0, s, a);            \
    else klaunch(k_pages_join<DD, TT, 128>, grid, 256, 0, s, a);                       \
  }
  JOIN(64, 0) JOIN(64, 1) JOIN(64, 2) JOIN(128, 0) JOIN(128, 1) JOIN(128, 2)
#undef JOIN
  return hipGetLastError();
}

}  // namespace moert
