// The 8-bit K/V cache of include/moert.h (moert_kv8_*): device view, index arithmetic and launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dev_math.h"

namespace moert {

constexpr int kKvBlock = 32;  // positions of a block
enum { KV_LEN = 0, KV_DROPPED = 1, KV_ARRIVED = 2, KV_STATE = 4 };  // words of a sequence's state

struct Kv8Dev {
  int seqs, kvh, d, slots, max_len;
  uint8_t *kc, *vc;
  float *ks, *vs;
  uint16_t *kt, *vt;
  uint32_t* bad;
  int* table;
  float* mass;
  int* state;
};

// moert_rows on the device; strides in elements.
struct KvRows {
  void* p;
  int f16;  // 0 f32, 1 fp16, 2 bf16 (of the paged cache only)
  long long seq, pos, head;
};

// Whether rows can be moved 16 bytes at a time.
inline int wide_rows(const KvRows& r) {
  const int m = r.f16 ? 8 : 4;
  return (uintptr_t)r.p % 16 == 0 && r.seq % m == 0 && r.pos % m == 0 && r.head % m == 0;
}

// Place of position t, element e in a block of V: what one lane multiplies at once, 8 positions of U = d / 16
// elements, is one run of bytes (k_kv8_attend says which lane).
template <int D>
__host__ __device__ __forceinline__ constexpr int v_place(int t, int e) {
  constexpr int U = D / 16;
  return ((e / U * 4 + t % 16 / 4) * U + e % U) * 8 + t % 4 + 4 * (t / 16);
}

__device__ __forceinline__ int kv_len(const Kv8Dev& c, int s) {
  const int n = c.state[(size_t)s * KV_STATE + KV_LEN];
  return n < 0 ? 0 : n > c.max_len ? c.max_len : n;
}
// A slot is used as an index only after this: whatever the table holds, it stays inside the buffers.
__device__ __forceinline__ int kv_slot(const Kv8Dev& c, int raw) {
  return (unsigned)raw < (unsigned)c.slots ? raw : 0;
}

struct KvAttnPlan {
  int splits;         // workgroups of a column tile along the cache, at most
  size_t tot, ml, parts, lse;  // offsets of the parts of the workspace
  size_t bytes;
};
KvAttnPlan kv8_attn_plan(const Kv8Dev& c, int n_seqs, int heads, int n, bool track);

hipError_t launch_kv8_clear(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs);
hipError_t launch_kv8_append(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, KvRows k, KvRows v, int n);
hipError_t launch_kv8_read(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int pos, int n, KvRows k, KvRows v);
hipError_t launch_kv8_evict(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int keep, int first, int last);
hipError_t launch_kv8_attend(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int heads, int n, float scale,
                             KvRows q, KvRows out, float decay, void* ws);

}  // namespace moert
