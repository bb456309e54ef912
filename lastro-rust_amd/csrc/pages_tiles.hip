// Attention of many rows over the paged 16-bit K/V cache (pages.h), on the matrix cores with f32 sums.
//
// A row is one query head at one position; the rows of a KV head's group, position by position, go in tiles of 128, 32
// to each of four waves. Per block of 32 positions of the cache, for 32 rows:
//   S = K Q^T    MFMA 32x32x16, rows = positions, columns = rows of the tile
//   softmax      p = 2^(S f - M), f = scale log2 e. M, the running maximum less 7, moves only where it has to (a weight
//                above 2^15), so most blocks cost no exchange between lanes and leave O alone.
//   O += V^T P^T MFMA 32x32x16, rows = elements. A lane of S holds, of its column, the positions 8 (r / 4) + 4 (lane / 32)
//                + r % 4, which is what it has to hold of P here when V's positions are taken in that order: V lies so in
//                the pool, and p never leaves its lane.
// Both operands of the cache lie in the pool as the matrix instructions take them, so 32 or 64 positions at a time go to LDS in
// straight copies of 16 bytes a lane, past the registers, while those before them are worked on.
//
// What bounds it, measured on one MI355X: the chip's power, between the matrix cores and the vector unit. 16384 positions,
// 8 KV heads of 64 with 3 query heads each, fp16, 825 GFLOP: 876 us, 941 TFLOP/s (on another such device 936 us, 881
// TFLOP/s), at 1.77 GHz, the matrix cores busy in 45% of the cycles and vector instructions issuing in 60% (a library
// product of 8192 x 8192 x 8192: 1070 TFLOP/s at 1.58 GHz, 70% and 28%). A block of 32 x 32 scores is 8 MFMAs of 32 cycles beside 48 vector instructions, 16 of them exponentials at
// half the rate, and 5 others. Measured on the way, same case: the maximum looked at in every block, through a second copy
// of the accumulators, 1084; two blocks a stage without it 916; copies by one base 888; two running sums, not four, 870. Two
// tiles of rows to a wave 956 for 934, priorities for the MFMAs or three stages in LDS within 1%.
#include <type_traits>

#include "pages_dev.h"

namespace moert {

namespace {

constexpr int kWaves = 4;

// Blocks of a stage, stages in LDS, and waves to a SIMD. Wide heads of 16 bits fit three waves with one block to a stage
// (twelve prompts of 128: 355 us, with two blocks and two waves 377); f32 would spill there.
template <int D, int T>
struct Shape {
  static constexpr bool kTight = D == 128 && T != PG_F32;
  static constexpr int kStage = kTight ? 1 : 2, kStages = kTight ? 3 : 2, kPerSimd = D == 64 || kTight ? 3 : 2;
};

template <int D, int T>
__global__ __launch_bounds__(kWaves * 64, (Shape<D, T>::kPerSimd)) void k_pages_tiles(PgArgs a) {
  constexpr int kStage = Shape<D, T>::kStage, NB = Shape<D, T>::kStages;
  constexpr int KS = D / 16, U = D / 32, W = 32 * kWaves, kBytes = 64 * D;  // of a block of K or V
  constexpr bool LO = T == PG_F32;  // queries and weights as two fp16
  __shared__ __align__(16) uint8_t lds[NB][kStage][2][kBytes];
  const PagesDev& c = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, G = lane >> 5;
  // the tiles of a KV head run on one XCD (workgroups go round them in turn) where there are eight of them
  const int id = blockIdx.x, h = id % c.kvh, split = id / c.kvh % a.splits, y = id / c.kvh / a.splits;
  PgTile t;
  if (!pg_tile(a, y, W, &t)) return;
  const int row1 = min(t.row0 + W, t.rows);
  const int seen = max(0, t.sees0 + (row1 - 1) / a.g), blocks = (seen + kPgBlock - 1) / kPgBlock;
  const int stages = (blocks + kStage - 1) / kStage, used = pg_tiles_used(a, blocks);
  if (split >= used) return;

  // this split's stages: split, split + used, ..; each wave copies a quarter of one. Lane x holds the place in the pool of
  // the wave's block of the x-th of 64
  constexpr int kPart = kStage * 2 * kBytes / kWaves, kCopies = kPart / 1024;
  const int* table = c.table + (size_t)t.s * c.max_pages;
  const int from = w * kPart, block_w = from / (2 * kBytes), in_w = from % kBytes, last = blocks - 1;
  const uint8_t* pool = (const uint8_t*)(from / kBytes % 2 ? c.v : c.k) + in_w;
  const uint32_t into = pg_lds(lds) + from;
  const int count = max(0, (stages - split + used - 1) / used);
  int place = 0;
  auto copy = [&](int x) {
    if (x % 64 == 0) {
      const int b = min((split + (x + lane) * used) * kStage + block_w, last);
      place = pg_block(c, pg_page(c, gmem(table)[b >> (c.lp - 5)]), h, b);
    }
    const uint8_t* src = pool + (size_t)__builtin_amdgcn_readlane(place, x % 64) * kBytes;
    pg_copy_to_lds<kCopies, false>(src, lane * 16, into + x % NB * (kStage * 2 * kBytes));
  };
#pragma unroll
  for (int x = 0; x < NB - 1; x++)
    if (x < count) copy(x);
  // the x-th stage's copies have come, from all waves, which are done with the one before; another one's set out
  auto arrive = [&](int x) {
    if (x + NB - 1 <= count) pg_wait_copies<(NB - 2) * kCopies>();
    else pg_wait_copies<0>();
    pg_wait_reads();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (x + NB - 1 < count) copy(x + NB - 1);
  };

  // queries, and the rows that the wave's columns see
  uint4 qh[KS], ql[LO ? KS : 1];
  const int mine = t.row0 + w * 32, row = min(mine + col, t.rows - 1), i = row / a.g, sees = t.sees0 + i;
  int qe = 0;
  {
    const long long at = (long long)(t.lo + i) * a.q.pos + (long long)(h * a.g + row % a.g) * a.q.head + G * 8;
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
      for (int k = 0; k < KS; k++) pg_split<T>(v[k], qe, &qh[k], &ql[k]);
    } else {
#pragma unroll
      for (int k = 0; k < KS; k++) qh[k] = pg_query16<T>(a, at + k * 16);
    }
  }
  const float f = pg_factor(a, qe);
  const bool idle = mine >= t.rows;
  const int least = t.sees0 + min(mine, t.rows - 1) / a.g;             // rows that the wave's first column sees
  const int most = idle ? 0 : t.sees0 + min(mine + 31, t.rows - 1) / a.g;  // and its last
  const int len = t.sees0 + t.rows / a.g - 1;                          // rows of the sequence

  float Sm = kPgNone, M = kPgNone, rest = 0.0f, l = 0.0f;  // the maximum as a sum of products, and times f; a lane's own sum
  pg_f16 O[U];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int x = 0; x < 16; x++) O[u][x] = 0.0f;

  auto scores = [&](const uint8_t* kp, pg_f16& S) {
#pragma unroll
    for (int x = 0; x < 16; x++) S[x] = 0.0f;
    uint4 ka[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) ka[k] = *reinterpret_cast<const uint4*>(kp + k * 1024 + lane * 16);
#pragma unroll
    for (int k = 0; k < KS; k++) {
      S = pg_mfma<T>(ka[k], qh[k], S);
      if constexpr (LO) S = pg_mfma<T>(ka[k], ql[k], S);
    }
  };
  // A block's weights; part takes their sums, two that do not wait for each other. Of 16 bits they are those of the rounded
  // ones, a pair to an instruction.
  auto weights = [&](auto far, const pg_f16& S, uint4* ph, uint4* pl, float* part) {
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float p[2];
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const float sc = S[s2 * 8 + j * 2 + z];
          p[z] = __builtin_amdgcn_exp2f(decltype(far)::value ? __builtin_fmaf(sc - Sm, f, rest) : __builtin_fmaf(sc, f, -M));
        }
        hi[j] = pg_pack<T>(p[0], p[1]);
        if constexpr (LO) {
          lo[j] = pg_rest<T>(hi[j], p[0], p[1]);
          part[0] += p[0];
          part[1] += p[1];
        } else {
          part[j % 2] = pg_add<T>(hi[j], part[j % 2]);
        }
      }
      ph[s2] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (LO) pl[s2] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  };
  // Moves the maximum to m. Weights are taken of S f - M, M rounded, and so is what they are multiplied by; far from 0,
  // where that rounding is more than a small part of a weight, of (S - Sm) f + 7: rest is 7 there, and otherwise Sm f - M.
  auto rescale = [&](float m) {
    const float to = __builtin_fmaxf(__builtin_fmaf(m, f, -kPgShift), kPgNone);  // finite where nothing is seen yet
    const bool far = __builtin_fabsf(to) > kPgFar;
    const float al = __builtin_amdgcn_exp2f(far ? (Sm - m) * f : M - to);
    Sm = m;
    M = to;
    rest = far ? kPgShift : __builtin_fmaf(m, f, -to);
    l *= al;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int x = 0; x < 16; x++) O[u][x] *= al;
  };
  auto is_far = [&](float m) { return __any(__builtin_fabsf(m * f) > kPgFar && m > kPgNone); };
  auto outputs = [&](auto masked, const uint8_t* vp, const uint4* ph, const uint4* pl, int b) {
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      uint32_t keep[4];  // memory behind the sequence's rows may hold anything, and 0 times that would be NaN
      if constexpr (decltype(masked)::value) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int at = b * kPgBlock + 16 * s2 + 4 * G + j % 2 * 2 + j / 2 * 8;
          keep[j] = (at < len ? 0xffffu : 0u) | (at + 1 < len ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        uint4 va = *reinterpret_cast<const uint4*>(vp + ((2 * s2 + G) * D + 32 * u + col) * 16);
        if constexpr (decltype(masked)::value)
          va = make_uint4(va.x & keep[0], va.y & keep[1], va.z & keep[2], va.w & keep[3]);
        O[u] = pg_mfma<T>(va, ph[s2], O[u]);
        if constexpr (LO) O[u] = pg_mfma<T>(va, pl[s2], O[u]);
      }
    }
  };

  // Stages that all columns of the wave see whole. Weights come before any maximum is looked at: only where their sum says
  // that one is above 2^15 or so, the maximum moves and they are taken again. Scores far from 0 are left to what follows.
  bool arrived = false;
  int x = 0, st = split;
  for (const int full = min(stages, max(least, 0) / (kStage * kPgBlock)); st < full; st += used, x++) {
    arrive(x);
    uint8_t(*at)[2][kBytes] = lds[x % NB];
    pg_f16 S[kStage];
    uint4 ph[kStage][2], pl[kStage][LO ? 2 : 1];
#pragma unroll
    for (int j = 0; j < kStage; j++) scores(at[j][0], S[j]);
    float part[2] = {0.0f, 0.0f};
    bool move = x == 0;  // there is no maximum yet
    if (!move) {
#pragma unroll
      for (int j = 0; j < kStage; j++) weights(std::false_type{}, S[j], ph[j], pl[j], part);
      move = __any(!(part[0] + part[1] <= 32768.0f));
    }
    if (move) {
      float m = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < kStage; j++)
#pragma unroll
        for (int x = 0; x < 16; x++) m = __builtin_fmaxf(m, S[j][x]);
      m = __builtin_fmaxf(Sm, max_stage<32>(m));
      if (is_far(m)) {
        arrived = true;
        break;
      }
      rescale(m);
      part[0] = part[1] = 0.0f;
#pragma unroll
      for (int j = 0; j < kStage; j++) weights(std::false_type{}, S[j], ph[j], pl[j], part);
    }
    l += part[0] + part[1];
#pragma unroll
    for (int j = 0; j < kStage; j++) outputs(std::false_type{}, at[j][1], ph[j], pl[j], 0);
  }
  // The others, and all that comes after scores far from 0: differences of scores before products.
  for (; st < stages; st += used, x++) {
    if (!arrived) arrive(x);
    uint8_t(*at)[2][kBytes] = lds[x % NB];
    arrived = false;
#pragma unroll 1
    for (int j = 0; j < kStage; j++) {
      const int b = st * kStage + j;
      if (b * kPgBlock >= most) break;
      pg_f16 S;
      uint4 ph[2], pl[LO ? 2 : 1];
      scores(at[j][0], S);
      float m = -__builtin_inff();
#pragma unroll
      for (int x = 0; x < 16; x++) {
        if (b * kPgBlock + 8 * (x / 4) + 4 * G + x % 4 >= sees) S[x] = -__builtin_inff();
        m = __builtin_fmaxf(m, S[x]);
      }
      m = __builtin_fmaxf(Sm, max_stage<32>(m));
      if (__any(m > Sm)) rescale(m);
      float part[2] = {0.0f, 0.0f};
      weights(std::true_type{}, S, ph, pl, part);
      l += part[0] + part[1];
      outputs(std::true_type{}, at[j][1], ph, pl, b);
    }
  }
  if (idle) return;
  l += partner<32>(l);
  if (mine + col >= t.rows) return;
  if (used == 1) {
    const float inv = sees > 0 ? 1.0f / l : 0.0f;
    const long long at = (long long)(t.lo + i) * a.out.pos + (long long)(h * a.g + row % a.g) * a.out.head + 4 * G;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float o[4] = {O[u][4 * r] * inv, O[u][4 * r + 1] * inv, O[u][4 * r + 2] * inv, O[u][4 * r + 3] * inv};
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
            pg_f4{O[u][4 * r], O[u][4 * r + 1], O[u][4 * r + 2], O[u][4 * r + 3]};
    if (G == 0) a.ml[wc] = make_float2(M, l);
  }
}

}  // namespace

hipError_t launch_pages_tiles(hipStream_t s, PgArgs a) {
  const unsigned grid = (unsigned)a.tiles * a.c.kvh * a.splits;
#define TILES(DD, TT) \
  if (a.c.d == DD && a.q.f16 == TT) klaunch(k_pages_tiles<DD, TT>, grid, kWaves * 64, 0, s, a);
  TILES(64, 0) TILES(64, 1) TILES(64, 2) TILES(128, 0) TILES(128, 1) TILES(128, 2)
#undef TILES
  return hipGetLastError();
}

}  // namespace moert
