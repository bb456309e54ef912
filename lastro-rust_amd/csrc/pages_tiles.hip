// Attention of many rows over the paged 16-bit K/V cache (pages.h), on the matrix cores with f32 sums.
//
// A row is one query head at one position; the rows of a KV head's group, position by position, go in tiles of 128 Q, 32 Q
// to each of four waves. Per block of 32 positions of the cache, for 32 rows:
//   S = K Q^T    MFMA 32x32x16, rows = positions, columns = rows of the tile
//   softmax      p = 2^(S f - M), f = scale log2 e. The running maximum M moves only where it has to (a weight above
//                2^8), so most blocks cost no exchange between lanes and leave O alone.
//   O += V^T P^T MFMA 32x32x16, rows = elements. A lane of S holds, of its column, the positions 8 (r / 4) + 4 (lane / 32)
//                + r % 4, which is what it has to hold of P here when V's positions are taken in that order: V lies so in
//                the pool, and p never leaves its lane.
// Both operands of the cache lie in the pool as the matrix instructions take them, so 64 positions at a time go to LDS in
// straight copies of 16 bytes a lane, past the registers, while the 64 before them are worked on.
#include <type_traits>

#include "pages_dev.h"

namespace moert {

namespace {

constexpr int kWaves = 4;
constexpr int kStage = 2;  // blocks staged together

// 16 bytes of each lane to LDS, in a row from `dst` (the wave's) on, without a way through registers. Not by the builtin:
// the compiler cannot tell the buffer that it fills from the one being read, and would wait for the copy before each read.
// Whoever reads them waits for vmcnt 0 and a barrier first.
__device__ __forceinline__ void pg_copy_to_lds(const uint8_t* src, uint8_t* dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(src) : "memory", "m0");
}

template <int D, int T, int Q>
__global__ __launch_bounds__(kWaves * 64, 2) void k_pages_tiles(PgArgs a) {
  constexpr int KS = D / 16, U = D / 32, W = 32 * Q * kWaves, kBytes = 64 * D;  // of a block of K or V
  constexpr bool LO = T == PG_F32;  // queries and weights as two fp16
  __shared__ __align__(16) uint8_t lds[2][kStage][2][kBytes];
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, G = lane >> 5;
  // the tiles of a KV head run on one XCD (workgroups go round them in turn) where there are eight of them, the last ones
  // of a sequence, which see the most, first
  const int id = blockIdx.x, h = id % c.kvh, split = id / c.kvh % a.splits, y = a.tiles - 1 - id / c.kvh / a.splits;
  PgTile t;
  if (!pg_tile(a, y, W, &t)) return;
  const int row1 = min(t.row0 + W, t.rows);
  const int seen = max(0, t.sees0 + (row1 - 1) / a.g), blocks = (seen + kPgBlock - 1) / kPgBlock;
  const int stages = (blocks + kStage - 1) / kStage, used = pg_tiles_used(a, blocks);
  if (split >= used) return;

  // queries, and the rows that each column sees
  uint4 qh[Q][KS], ql[Q][LO ? KS : 1];
  float f[Q];
  int sees[Q];
  const int mine = t.row0 + w * 32 * Q;  // the wave's first row
#pragma unroll
  for (int x = 0; x < Q; x++) {
    const int row = min(mine + x * 32 + col, t.rows - 1), i = row / a.g;
    sees[x] = t.sees0 + i;
    const long long at = (long long)(t.lo + i) * a.q.pos + (long long)(h * a.g + row % a.g) * a.q.head + G * 8;
    int qe = 0;
    if constexpr (LO) {
      float v[KS][8], m = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        pg_query<T>(a, at + k * 16, v[k]);
#pragma unroll
        for (int j = 0; j < 8; j++) m = __builtin_fmaxf(m, __builtin_fabsf(v[k][j]));
      }
      qe = pg_split_exp(max_stage<32>(m));
#pragma unroll
      for (int k = 0; k < KS; k++) pg_split<T>(v[k], qe, &qh[x][k], &ql[x][k]);
    } else {
#pragma unroll
      for (int k = 0; k < KS; k++) qh[x][k] = pg_query16<T>(a, at + k * 16);
    }
    f[x] = pg_factor(a, qe);
  }
  const int least = t.sees0 + min(mine, t.rows - 1) / a.g;                     // rows that the wave's first column sees
  const int most = t.sees0 + min(mine + 32 * Q - 1, t.rows - 1) / a.g;         // and its last
  const bool idle = mine >= t.rows;
  const int len = t.sees0 + t.rows / a.g - 1;  // rows of the sequence

  float Sm[Q], M[Q], l[Q];  // the maximum as a sum of products, and times f; a lane's own sum
  pg_f16 O[Q][U];
#pragma unroll
  for (int x = 0; x < Q; x++) {
    Sm[x] = kPgNone;
    M[x] = kPgNone;
    l[x] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < 16; i++) O[x][u][i] = 0.0f;
  }
  bool far = false;
  float none = -__builtin_inff();
  asm("" : "+s"(none));

  // this split's stages: split, split + used, ..
  const int* table = c.table + (size_t)t.s * c.max_pages;
  const int block_w = w >> 1, last = blocks - 1, lb = c.lp - 5;
  const uint16_t* pool = w & 1 ? c.v : c.k;
  // wave w copies K (even) or V (odd) of block w / 2 of a stage
  auto page_of = [&](int st) { return pg_page(c, gmem(table)[min(st * kStage + block_w, last) >> lb]); };
  auto stage = [&](int st, int buf, int page) {
    const int b = min(st * kStage + block_w, last);
    const uint8_t* src = (const uint8_t*)(pool + (size_t)pg_block(c, __builtin_amdgcn_readfirstlane(page), h, b) *
                                                     (kPgBlock * D));
    uint8_t* dst = &lds[buf][block_w][w & 1][0];
#pragma unroll
    for (int i = 0; i < kBytes / 1024; i++)
      pg_copy_to_lds(src + i * 1024 + lane * 16, dst + i * 1024);
  };

  auto block = [&](auto masked, const uint8_t* kp, const uint8_t* vp, int b) {
    constexpr bool MASKED = decltype(masked)::value;
    pg_f16 S[Q];
#pragma unroll
    for (int x = 0; x < Q; x++)
#pragma unroll
      for (int i = 0; i < 16; i++) S[x][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const uint4 ka = *reinterpret_cast<const uint4*>(kp + k * 1024 + lane * 16);
#pragma unroll
      for (int x = 0; x < Q; x++) {
        S[x] = pg_mfma<T>(ka, qh[x][k], S[x]);
        if constexpr (LO) S[x] = pg_mfma<T>(ka, ql[x][k], S[x]);
      }
    }
    if constexpr (MASKED) {
#pragma unroll
      for (int x = 0; x < Q; x++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (b * kPgBlock + 8 * (i / 4) + 4 * G + i % 4 >= sees[x]) S[x][i] = -__builtin_inff();
    }
    float mx[Q];
    bool move = false;
#pragma unroll
    for (int x = 0; x < Q; x++) {
      mx[x] = none;
#pragma unroll
      for (int i = 0; i < 16; i++) mx[x] = __builtin_fmaxf(mx[x], S[x][i]);
      move |= __builtin_fmaf(mx[x], f[x], -M[x]) > kPgSlack;
    }
    if (__any(move)) {
#pragma unroll
      for (int x = 0; x < Q; x++) {
        const float m = __builtin_fmaxf(Sm[x], max_stage<32>(mx[x]));
        const float al = __builtin_amdgcn_exp2f((Sm[x] - m) * f[x]);
        Sm[x] = m;
        M[x] = __builtin_fmaxf(m * f[x], kPgNone);  // finite where nothing is seen yet
        far |= __any(__builtin_fabsf(M[x]) > kPgFar && m > kPgNone);
        l[x] *= al;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) O[x][u][i] *= al;
      }
    }
    uint4 ph[Q][2], pl[Q][LO ? 2 : 1];
    auto weights = [&](auto is_far) {
#pragma unroll
      for (int x = 0; x < Q; x++)
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float p[2];
#pragma unroll
            for (int z = 0; z < 2; z++) {
              const float sc = S[x][s2 * 8 + j * 2 + z];
              p[z] = __builtin_amdgcn_exp2f(decltype(is_far)::value ? (sc - Sm[x]) * f[x]
                                                                    : __builtin_fmaf(sc, f[x], -M[x]));
              l[x] += p[z];
            }
            hi[j] = pg_pack<T>(p[0], p[1]);
            if constexpr (LO) {
              const pg_f2 back = pg_unpack<T>(hi[j]);
              lo[j] = pg_pack<T>(p[0] - back.x, p[1] - back.y);
            }
          }
          ph[x][s2] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (LO) pl[x][s2] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    };
    if (far) weights(std::true_type{});
    else weights(std::false_type{});
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      uint32_t keep[4];  // memory behind the sequence's rows may hold anything, and 0 times that would be NaN
      if constexpr (MASKED) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int at = b * kPgBlock + 16 * s2 + 4 * G + j % 2 * 2 + j / 2 * 8;
          keep[j] = (at < len ? 0xffffu : 0u) | (at + 1 < len ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        uint4 va = *reinterpret_cast<const uint4*>(vp + ((2 * s2 + G) * D + 32 * u + col) * 16);
        if constexpr (MASKED) va = make_uint4(va.x & keep[0], va.y & keep[1], va.z & keep[2], va.w & keep[3]);
#pragma unroll
        for (int x = 0; x < Q; x++) {
          O[x][u] = pg_mfma<T>(va, ph[x][s2], O[x][u]);
          if constexpr (LO) O[x][u] = pg_mfma<T>(va, pl[x][s2], O[x][u]);
        }
      }
    }
  };

  if (blocks > 0) {
    int page = page_of(split);
    stage(split, 0, page);
    page = page_of(split + used);
    for (int st = split, buf = 0; st < stages; st += used, buf ^= 1) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the stage has come
      __syncthreads();
      if (st + used < stages) stage(st + used, buf ^ 1, page);
      page = page_of(st + 2 * used);
#pragma unroll 1
      for (int j = 0; j < kStage; j++) {
        const int b = st * kStage + j;
        if (!idle && b * kPgBlock < most) {
          if ((b + 1) * kPgBlock > least) block(std::true_type{}, lds[buf][j][0], lds[buf][j][1], b);
          else block(std::false_type{}, lds[buf][j][0], lds[buf][j][1], b);
        }
      }
    }
  }
  if (idle) return;
#pragma unroll
  for (int x = 0; x < Q; x++) {
    const int row = mine + x * 32 + col;
    const float sum = l[x] + partner<32>(l[x]);
    if (row >= t.rows) continue;
    const int i = row / a.g;
    if (used == 1) {
      const float inv = sees[x] > 0 ? 1.0f / sum : 0.0f;
      const long long at = (long long)(t.lo + i) * a.out.pos + (long long)(h * a.g + row % a.g) * a.out.head + 4 * G;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float o[4] = {O[x][u][4 * r] * inv, O[x][u][4 * r + 1] * inv, O[x][u][4 * r + 2] * inv,
                              O[x][u][4 * r + 3] * inv};
          pg_store<T, 4>(a, at + 32 * u + 8 * r, o);
        }
    } else {
      const size_t wc = (((size_t)h * a.tiles + y) * W + (row - t.row0)) * a.splits + split;
      float* po = a.part + wc * D + 4 * G;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          *reinterpret_cast<pg_f4*>(po + 32 * u + 8 * r) =
              pg_f4{O[x][u][4 * r], O[x][u][4 * r + 1], O[x][u][4 * r + 2], O[x][u][4 * r + 3]};
      if (G == 0) a.ml[wc] = make_float2(M[x], sum);
    }
  }
}

}  // namespace

hipError_t launch_pages_tiles(hipStream_t s, PgArgs a) {
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * a.splits;
#define TILES(DD, TT) \
  if (a.c.d == DD && a.q.f16 == TT) klaunch(k_pages_tiles<DD, TT, 1>, grid, kWaves * 64, 0, s, a);
  TILES(64, 0) TILES(64, 1) TILES(64, 2) TILES(128, 0) TILES(128, 1) TILES(128, 2)
#undef TILES
  return hipGetLastError();
}

}  // namespace moert
