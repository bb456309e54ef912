// Attention over the 8-bit K/V cache (kv8.h). A simple form: a wave per position and query head goes through the rows
// block by block, 32 scores at a time (lane t: row t), with a running maximum and sum; then each lane takes its
// elements of the output. The weights of the blocks for the mass: log2 of each block's sum by column (a column is one
// query head at one position), and of the column's whole sum; k_kv8_mass adds them up in order.
#include "kv8.h"
#include "launch.h"

namespace moert {

namespace {

constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float q_elem(const KvRows& r, long long at) {
  return r.f16 ? h2f(gmem((const uint16_t*)r.p)[at]) : gmem((const float*)r.p)[at];
}

template <int D>
__global__ __launch_bounds__(64) void k_kv8_simple(Kv8Dev c, KvRows q, KvRows out, int seq0, int heads, int n,
                                                   float scale, float* __restrict__ lse, float* __restrict__ tot) {
  __shared__ float Q[D], P[kKvBlock];
  const int g = heads / c.kvh, lane = threadIdx.x;
  const int hq = blockIdx.x % heads, i = blockIdx.x / heads, sc = blockIdx.y, s = seq0 + sc, h = hq / g;
  const int len = kv_len(c, s), sees = len - n + 1 + i;
  const size_t head = (size_t)s * c.kvh + h;
  const size_t col = ((size_t)sc * c.kvh + h) * n * g + (size_t)i * g + hq % g;
  for (int e = lane; e < D; e += 64) Q[e] = q_elem(q, sc * q.seq + i * q.pos + hq * q.head + e);
  __syncthreads();
  float m = -1e30f, l = 0.0f, o[D / 64] = {};
  const uint32_t bad = c.bad[head];
  for (int b = 0; b * kKvBlock < sees; b++) {
    const bool tail = b == len / kKvBlock;
    const size_t slot = head * c.slots + kv_slot(c, c.table[head * c.slots + b]);
    const float ks = tail ? 1.0f : c.ks[slot], vs = tail ? 1.0f : c.vs[slot];
    const int t = lane % kKvBlock;
    const bool in = b * kKvBlock + t < sees;
    float x = 0.0f;
    for (int e = 0; e < D; e++) {
      const float k = tail ? h2f(c.kt[head * kKvBlock * D + t * D + e])
                           : (float)((int)c.kc[slot * (kKvBlock * D) + t * D + e] - 128);
      x = __builtin_fmaf(Q[e], k, x);
    }
    x = x * (ks * (scale * kLog2e)) + 0.0f * vs;  // a block whose V is not finite has no weights either
    if (tail && (bad >> t & 1)) x = __int_as_float(0x7fc00000);
    const float mn = __builtin_fmaxf(m, group_max(in && x == x ? x : -1e30f)), a = __builtin_amdgcn_exp2f(m - mn);
    const float p = in ? __builtin_amdgcn_exp2f(x - mn) : 0.0f;
    const float sum = group_sum<32>(p);
    m = mn;
    l = __builtin_fmaf(l, a, sum);
    if (lse && lane == 0) lse[col * c.slots + b] = __builtin_amdgcn_logf(sum) + m;
    if (lane < kKvBlock) P[t] = p;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < D / 64; j++) {
      float y = 0.0f;
      for (int t = 0; t < kKvBlock && b * kKvBlock + t < sees; t++) {
        const int at = v_place<D>(t, j * 64 + lane);
        const float v = tail ? h2f(c.vt[head * kKvBlock * D + at])
                             : (float)((int)c.vc[slot * (kKvBlock * D) + at] - 128);
        y = __builtin_fmaf(P[t], v, y);
      }
      o[j] = __builtin_fmaf(o[j], a, y * vs);
    }
    __syncthreads();
  }
  for (int j = 0; j < D / 64; j++) {
    const float y = l == 0.0f ? 0.0f : o[j] / l;
    const long long at = sc * out.seq + i * out.pos + hq * out.head + j * 64 + lane;
    if (out.f16) ((uint16_t*)out.p)[at] = f2h(y);
    else ((float*)out.p)[at] = y;
  }
  if (tot && lane == 0) tot[col] = l == 0.0f ? __int_as_float(0x7f800000) : __builtin_amdgcn_logf(l) + m;
}

// mass = decay * mass + the block's weights, a thread per block.
__global__ void k_kv8_mass(Kv8Dev c, int seq0, int g, int n, float decay, const float* __restrict__ lse,
                           const float* __restrict__ tot) {
  const int sc = blockIdx.z, h = blockIdx.y, s = seq0 + sc, b = blockIdx.x * blockDim.x + threadIdx.x;
  const int len = kv_len(c, s);
  if (b * kKvBlock >= len) return;
  const size_t head = (size_t)s * c.kvh + h, col0 = ((size_t)sc * c.kvh + h) * n * g;
  float w = 0.0f;
  for (int i = 0; i < n; i++) {
    if (b * kKvBlock >= len - n + 1 + i) continue;
    for (int j = 0; j < g; j++) {
      const size_t col = col0 + (size_t)i * g + j;
      w += __builtin_amdgcn_exp2f(lse[col * c.slots + b] - tot[col]);
    }
  }
  float* m = c.mass + head * c.slots + kv_slot(c, c.table[head * c.slots + b]);
  *m = __builtin_fmaf(decay, *m, w);
}

}  // namespace

KvAttnPlan kv8_attn_plan(const Kv8Dev& c, int n_seqs, int heads, int n, bool track) {
  KvAttnPlan p;
  const size_t cols = (size_t)n_seqs * heads * n;
  p.splits = 1;
  p.parts = 0;
  p.lse = (cols * 4 + 255) / 256 * 256;
  p.bytes = p.lse + (track ? cols * c.slots * 4 : 0);
  return p;
}

hipError_t launch_kv8_attend(hipStream_t s, const Kv8Dev& c, int seq0, int n_seqs, int heads, int n, float scale,
                             KvRows q, KvRows out, float decay, void* ws) {
  const bool track = decay >= 0.0f;
  const KvAttnPlan p = kv8_attn_plan(c, n_seqs, heads, n, track);
  float* tot = track ? (float*)ws : nullptr;
  float* lse = track ? (float*)((char*)ws + p.lse) : nullptr;
  if (c.d == 64) klaunch(k_kv8_simple<64>, dim3(n * heads, n_seqs), 64, 0, s, c, q, out, seq0, heads, n, scale, lse, tot);
  else klaunch(k_kv8_simple<128>, dim3(n * heads, n_seqs), 64, 0, s, c, q, out, seq0, heads, n, scale, lse, tot);
  if (track)
    klaunch(k_kv8_mass, dim3((c.slots + 255) / 256, c.kvh, n_seqs), 256, 0, s, c, seq0, heads / c.kvh, n, decay, lse,
            tot);
  return hipGetLastError();
}

}  // namespace moert
