// What both attention kernels of the paged cache share (pages.h): types, queries, outputs, which rows a workgroup has.
#pragma once
#include <math.h>

#include "launch.h"
#include "pages.h"

namespace moert {

// Types of rows.
enum { PG_F32 = 0, PG_F16 = 1, PG_BF16 = 2 };

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_b2 __attribute__((ext_vector_type(2)));
typedef float pg_f2 __attribute__((ext_vector_type(2)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));

constexpr float kPgNone = -3.4e38f;  // maximum of what has no score yet; finite, so that differences with it are
// Weights are 2^7 for the maximum that they are taken of, which moves only for weights above 2^15: fp16 has 11 bits for them
// down to 2^-21 of the largest, and stops at 2^-31.
constexpr float kPgShift = 7.0f, kPgSlack = 15.0f;
constexpr float kPgFar = 1048576.0f;  // scores beyond it lose 2^-5 in a product less a maximum: differences come first
constexpr int kPgMaxSplits = 64;     // one lane each in the combine
constexpr float kPgLog2e = 1.44269504088896341f;

template <int T>
__device__ __forceinline__ uint32_t pg_pack(float a, float b) {
  const pg_f2 x = {a, b};
  if constexpr (T == PG_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, pg_b2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, pg_h2));
}
// What rounding to the pair `w` has left of a and b, as a pair.
template <int T>
__device__ __forceinline__ uint32_t pg_rest(uint32_t w, float a, float b) {
  if constexpr (T == PG_BF16) {
    return pg_pack<T>(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
  } else {
    const pg_h2 h = __builtin_bit_cast(pg_h2, w);
    return pg_pack<T>(a - (float)h.x, b - (float)h.y);
  }
}

// x + a pair's sum.
template <int T>
__device__ __forceinline__ float pg_add(uint32_t w, float x) {
  if constexpr (T == PG_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pg_b2, w), pg_b2{(__bf16)1.0f, (__bf16)1.0f}, x, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pg_h2, w), pg_h2{(_Float16)1.0f, (_Float16)1.0f}, x, false);
}

// D = A B + C on the matrix cores, A and B in 16 bits, 8 elements of a lane each.
template <int T>
__device__ __forceinline__ pg_f4 pg_mfma(uint4 a, uint4 b, pg_f4 c) {
  if constexpr (T == PG_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_b8, a), __builtin_bit_cast(pg_b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_h8, a), __builtin_bit_cast(pg_h8, b), c, 0, 0, 0);
}
template <int T>
__device__ __forceinline__ pg_f16 pg_mfma(uint4 a, uint4 b, pg_f16 c) {
  if constexpr (T == PG_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pg_b8, a), __builtin_bit_cast(pg_b8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pg_h8, a), __builtin_bit_cast(pg_h8, b), c, 0, 0, 0);
}

struct PgArgs {
  PagesDev c;
  KvRows q, out;
  const int* starts;
  int tokens, g, splits, tiles;  // g: query heads to a KV head
  int least, most;  // sequences of so many rows are attended
  int vec;          // bit 0: q can be loaded 16 bytes at a time, bit 1: out can be stored so
  float kf;         // |scale| log2 e, less 2^ke
  int ke;
  uint32_t sign;    // of the scale
  float* part;      // [KV head][tile][row of it][split][D]
  float2* ml;       // [KV head][tile][row of it][split]: maximum, sum
};

// Eight elements of a query from element `at` on, of a scale's sign.
template <int T>
__device__ __forceinline__ void pg_query(const PgArgs& a, long long at, float* x) {
  if constexpr (T == PG_F32) {
    const float* p = (const float*)a.q.p + at;
    if (a.vec & 1) {
      const float4 u = gload_f4(p), v = gload_f4(p + 4);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = gmem(p)[j];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __uint_as_float(__float_as_uint(x[j]) ^ a.sign);
  }
}
template <int T>
__device__ __forceinline__ uint4 pg_query16(const PgArgs& a, long long at) {
  const uint16_t* p = (const uint16_t*)a.q.p + at;
  uint32_t w[4];
  if (a.vec & 1) {
    const uint4 v = gload_u4(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (uint32_t)gmem(p)[2 * j] | (uint32_t)gmem(p)[2 * j + 1] << 16;
  }
  const uint32_t flip = a.sign ? 0x80008000u : 0u;
  return make_uint4(w[0] ^ flip, w[1] ^ flip, w[2] ^ flip, w[3] ^ flip);
}

// N KB (a multiple of 4) of memory to LDS, 16 bytes of each lane at a time, without a way through registers; `src` and
// `dst` (a place in LDS) are the wave's, `lane` 16 times the lane. The instruction's offset counts on both sides. Not by the builtin: the
// compiler cannot tell the buffer that is filled from the one being read, and would wait for the copy before each read.
// Whoever reads them waits by pg_wait_copies<M> first: for all but the last M copies and loads of the wave (loads of the
// compiler's among them only make it wait for more). STREAM: with the non-temporal hint.
template <int N, bool STREAM>
__device__ __forceinline__ void pg_copy_to_lds(const uint8_t* src, uint32_t lane, uint32_t dst) {
  if constexpr (N > 4) {
    pg_copy_to_lds<4, STREAM>(src, lane, dst);
    pg_copy_to_lds<N - 4, STREAM>(src + 4096, lane, dst + 4096);
  } else {
    static_assert(N == 4, "");
    dst = __builtin_amdgcn_readfirstlane(dst);
#define PG_COPY(HINT)                                                                                        \
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" HINT                        \
               "\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" HINT                                          \
               "\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4" HINT                                          \
               "\n\tglobal_load_lds_dwordx4 %1, %2 offset:%5" HINT                                          \
               : : "s"(dst), "v"(lane), "s"(src), "n"(1 * 1024), "n"(2 * 1024), "n"(3 * 1024) : "memory", "m0");
    if constexpr (STREAM) {
      PG_COPY(" nt")
    } else {
      PG_COPY("")
    }
#undef PG_COPY
  }
}
// A place in LDS as a copy takes it.
__device__ __forceinline__ uint32_t pg_lds(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
template <int N>
__device__ __forceinline__ void pg_wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// The wave's reads of LDS have their data: copies may go over what they read.
__device__ __forceinline__ void pg_wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// f32 queries enter as two fp16: their row by a power of two to below 2^10, then what the first rounding leaves. So they
// are off by 2^-22 of themselves, or by half of fp16's least step, 2^-34 of the row's largest. pg_split_exp: log2 of what the row has been divided by; m: its largest magnitude.
__device__ __forceinline__ int pg_split_exp(float m) {
  return (m > 0.0f && m < __int_as_float(0x7f800000) ? __builtin_amdgcn_frexp_expf(m) : 0) - 10;
}
template <int T>
__device__ __forceinline__ void pg_split(const float* x, int e, uint4* hi, uint4* lo) {
  const int e1 = -e / 2, e2 = -e - e1;  // in two factors: either alone could leave the type
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float p = __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(x[2 * j], e1), e2);
    const float q = __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(x[2 * j + 1], e1), e2);
    h[j] = pg_pack<T>(p, q);
    l[j] = pg_rest<T>(h[j], p, q);
  }
  *hi = make_uint4(h[0], h[1], h[2], h[3]);
  *lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// What a sum of products is multiplied by. Never 0: what is masked has to stay -inf, and f32's smallest number, 2^-149, of a
// sum below 10^38 is no score. Nor infinite, where it leaves f32 without the scores (of keys that are small): sums that differ
// do so by 2^-58 or more there, and 2^127 of that is all the weight or none, as more of it would be.
__device__ __forceinline__ float pg_factor(const PgArgs& a, int qe) {
  return __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_ldexpf(a.kf, a.ke + qe), 0x1p-149f), 0x1p127f);
}

// An output is a mean of fp16 values: what roundings bring beyond the largest of them is cut.
template <int T>
__device__ __forceinline__ float pg_clip(float x) {
  if constexpr (T == PG_F16) return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x;
  return x;
}

// N (4 or 8) elements of an output from element `at` on.
template <int T, int N>
__device__ __forceinline__ void pg_store(const PgArgs& a, long long at, const float* x) {
  if constexpr (T == PG_F32) {
    float* p = (float*)a.out.p + at;
    if (a.vec & 2) {
#pragma unroll
      for (int j = 0; j < N; j += 4) *reinterpret_cast<pg_f4*>(p + j) = pg_f4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) p[j] = x[j];
    }
  } else {
    uint16_t* p = (uint16_t*)a.out.p + at;
    uint32_t w[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; j++) w[j] = pg_pack<T>(pg_clip<T>(x[2 * j]), pg_clip<T>(x[2 * j + 1]));
    if (a.vec & 2) {
      if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) p[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Tiles of W rows (a row: one query head of the group at one position, position by position) in a packed batch: those of
// sequence s are counted from floor(starts[s] g / W) + s on, which leaves room for all of them, the last not full one
// too, without anybody adding up. So tile y is the sequence's that is the last to begin at or before y: 64 candidates at
// a time, one to a lane.
__device__ __forceinline__ int pg_first_tile(const PgArgs& a, int s, int w) {
  return min(max(gmem(a.starts)[s], 0), a.tokens) * a.g / w + s;
}
__device__ __forceinline__ int pg_find(const PgArgs& a, int y, int w) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = a.c.seqs;
  while (len > 1) {
    const int step = (len + 63) / 64, i = lane * step;
    const bool in = i < len && pg_first_tile(a, lo + min(i, len - 1), w) <= y;
    const unsigned long long m = __ballot(in);
    const int x = m ? 63 - __builtin_clzll(m) : 0;
    lo += x * step;
    len = min(step, len - x * step);
  }
  return lo;
}

// What a tile has to do.
struct PgTile {
  int s, row0, rows, lo;  // sequence, its first row, rows of the sequence, place of the sequence in the batch
  int sees0;              // rows that the sequence's first position sees
};
__device__ __forceinline__ bool pg_tile(const PgArgs& a, int y, int w, PgTile* t) {
  int s, first;
  if (a.most > 1) {
    s = pg_find(a, y, w);
    first = pg_first_tile(a, s, w);
  } else {  // one position of each sequence
    const int per = (a.g + w - 1) / w;
    s = y / per;
    first = s * per;
  }
  const int2 span = pg_span(a.starts, s, a.tokens);
  const int n = span.y - span.x;
  t->s = s;
  t->lo = span.x;
  t->rows = n * a.g;
  // Sequences in the batch's order, of each the last tiles, which see the most, first. Where the longest prompts come first
  // too, no long tile is begun late: 30.9 us, the shortest first 32.4 (geometric mean of 64 batches).
  const int tiles = (t->rows + w - 1) / w, at = tiles - 1 - (y - first);
  t->row0 = at * w;
  t->sees0 = pg_seen(a.c, s) - n + 1;
  // starts that do not begin at 0, or fall, leave tiles before the sequence's first
  return n >= a.least && n <= a.most && at >= 0 && at < tiles;
}
// Tiles that a batch may have.
inline int pg_tiles(const PgArgs& a, int w) {
  return a.most > 1 ? (int)((long long)a.tokens * a.g / w) + a.c.seqs : a.c.seqs * ((a.g + w - 1) / w);
}

// Splits of a tile of 128 rows that have work, of `blocks` blocks.
__device__ __forceinline__ int pg_tiles_used(const PgArgs& a, int blocks) {
  return max(1, min(a.splits, (blocks + 7) / 8));
}

// a.tiles and a.splits say how; launch_pages_join joins the splits of tiles of `width` rows.
hipError_t launch_pages_tiles(hipStream_t s, PgArgs a);
hipError_t launch_pages_cols(hipStream_t s, PgArgs a);
hipError_t launch_pages_join(hipStream_t s, PgArgs a, int width);

}  // namespace moert
