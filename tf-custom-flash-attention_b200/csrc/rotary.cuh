// Query/key head norms with the position rotation, and the write of new keys
// and values into the paged cache, which applies them on the way.
//
//   n = x * rsqrt(mean(x^2) + eps)           (per head; skipped without a weight)
//   y = R(pos) (n * w)                       R turns feature pairs by pos * base^(-2i/rot)
// Backward: g = R(pos)^T dy,  dw = sum g * n,  dx = rsqrt(..) * (g w - n * mean(g w n)).
//
// Bound: HBM bytes (forward: x in, y out; backward: x, dy in, dx out); per
// element ~10 fp32 operations.  One group of LANES lanes owns one head row,
// eight features a lane, so the row's sum is three or four shuffles and both
// members of every rotated pair sit in one lane: for pairs (i, i + rot/2) a lane
// holds features 4j.. and rot/2 + 4j.., for neighbouring pairs 8j..8j+7.  A
// group walks several heads of one token with the token's cosines and sines in
// registers, four heads at a time (eight loads in flight a lane).
// All arithmetic is fp32, rounded to T once, at the store.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace sdpa_b200 {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kHeads = 4;        // heads a group has in flight
constexpr int kGradBlocks = 592; // most token blocks of the backward (rows of its workspace)

// One of q, k (or v, copied as it is).
struct Stream {
  const void* x;         // [tokens, heads, D], row stride `stride` elements a token
  const void* dy;        // backward
  void* y;               // dense [tokens, heads, D] (backward: dx); null: written to the cache
  const void* weight;    // [D] or null (no norm)
  const int* positions;  // [tokens] or null: token % period
  int64_t stride, dy_stride;
  int tokens, heads, period;
};

struct Params {
  Stream q, k, v;
  int D, D_v;
  int weight_f32;      // weights are float32 (else T)
  float eps;
  const float* table;  // [max_positions, rot]: cos | sin; null: no rotation
  int max_positions, rot, interleaved;
  // cache write
  PagedView view;
  void* k_pages;
  void* v_pages;
  // backward
  float* partial;      // [blocks, 2, D]
  void* dw_q;
  void* dw_k;
  int blocks;
};

template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
  using type = float4;
  static __device__ __forceinline__ void unpack(const float4& r, float* x) { x[0] = r.x, x[1] = r.y, x[2] = r.z, x[3] = r.w; }
  static __device__ __forceinline__ float4 pack(const float* x) { return make_float4(x[0], x[1], x[2], x[3]); }
};
template <>
struct Vec4<__half> {
  using type = uint2;
  static __device__ __forceinline__ void unpack(const uint2& r, float* x) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
  static __device__ __forceinline__ uint2 pack(const float* x) {
    return make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
  }
};

// Where a lane's eight features lie and how they turn.
struct Place {
  int a, b;           // first feature of its two groups of four
  bool live, turned;  // inside the row; inside the rotated part
};
__device__ __forceinline__ Place place_of(int lane, const Params& p) {
  Place c;
  c.live = lane * 8 < p.D;
  c.turned = p.table && lane * 8 < p.rot;
  const bool halves = c.turned && !p.interleaved;
  c.a = halves ? lane * 4 : lane * 8;
  c.b = halves ? p.rot / 2 + lane * 4 : lane * 8 + 4;
  return c;
}

template <typename T>
__device__ __forceinline__ void load_weight(const void* w, int f32, const Place& c, float* out) {
  if (!w || !c.live) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = 1.0f;
    return;
  }
  if (f32) {
    const float* f = static_cast<const float*>(w);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = f[c.a + e], out[4 + e] = f[c.b + e];
  } else {
    const T* f = static_cast<const T*>(w);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = to_f<T>(f[c.a + e]), out[4 + e] = to_f<T>(f[c.b + e]);
  }
}

// Cosines and sines of a lane's four pairs at `pos` (1 and 0 where nothing turns).
__device__ __forceinline__ void load_turn(const Params& p, const Place& c, int lane, int64_t pos, float* cs, float* sn) {
#pragma unroll
  for (int e = 0; e < 4; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
  if (!p.table) return;
  if (pos < 0 || pos >= p.max_positions) {
    if (lane == 0) atomicOr(&g_status_word, kStatusBadIndex);
    pos = pos < 0 ? 0 : p.max_positions - 1;
  }
  if (c.turned) {
    const float* row = p.table + pos * p.rot + lane * 4;
    const float4 a = __ldg(reinterpret_cast<const float4*>(row));
    const float* srow = row + p.rot / 2;
    const float4 b = __ldg(reinterpret_cast<const float4*>(srow));
    cs[0] = a.x, cs[1] = a.y, cs[2] = a.z, cs[3] = a.w;
    sn[0] = b.x, sn[1] = b.y, sn[2] = b.z, sn[3] = b.w;
  }
}

// x <- R x (sign = 1) or R^T x (sign = -1) on a lane's eight features.
__device__ __forceinline__ void turn(float* x, const float* cs, const float* sn, bool interleaved, float sign) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = x[2 * e], b = x[2 * e + 1], s = sign * sn[e];
      x[2 * e] = a * cs[e] - b * s;
      x[2 * e + 1] = b * cs[e] + a * s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = x[e], b = x[4 + e], s = sign * sn[e];
      x[e] = a * cs[e] - b * s;
      x[4 + e] = b * cs[e] + a * s;
    }
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float x, unsigned mask) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1) x += __shfl_xor_sync(mask, x, d);
  return x;
}

// Heads [h0, h0 + kHeads) of one token's row: norm, rotation, store.
template <typename T, int LANES>
__device__ __forceinline__ void forward_heads(const T* x, T* y, int heads, int h0, const Params& p, const Place& c,
                                              const float* w, bool norm, const float* cs, const float* sn,
                                              unsigned mask) {
  using V = Vec4<T>;
  typename V::type ra[kHeads], rb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (c.live && h0 + i < heads) {
      ra[i] = __ldg(reinterpret_cast<const typename V::type*>(x + (h0 + i) * p.D + c.a));
      rb[i] = __ldg(reinterpret_cast<const typename V::type*>(x + (h0 + i) * p.D + c.b));
    }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (h0 + i >= heads) break;  // the same for every lane of the group
    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (c.live) V::unpack(ra[i], f), V::unpack(rb[i], f + 4);
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
      const float r = rsqrtf(group_sum<LANES>(ss, mask) / static_cast<float>(p.D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= r * w[e];
    }
    turn(f, cs, sn, p.interleaved, 1.0f);
    if (c.live) {
      *reinterpret_cast<typename V::type*>(y + (h0 + i) * p.D + c.a) = V::pack(f);
      *reinterpret_cast<typename V::type*>(y + (h0 + i) * p.D + c.b) = V::pack(f + 4);
    }
  }
}

// Token t of one stream: the head groups u of [u0, units) this block row takes.
template <int LANES>
struct Group {
  int lane;
  unsigned mask;
  int64_t token;
  __device__ __forceinline__ Group() {
    lane = threadIdx.x % LANES;
    mask = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES));
    token = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  }
};

// grid.x: blocks of kThreads / LANES tokens; grid.y: shares of a token's head
// groups (more of them when there are few tokens).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Params p) {
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place c = place_of(g.lane, p);
  pdl_wait();
  const int uq = (p.q.heads + kHeads - 1) / kHeads, uk = (p.k.heads + kHeads - 1) / kHeads;
  const int64_t tokens = max(p.q.tokens, p.k.tokens);
  if (g.token >= tokens) return;
  float cs[4], sn[4], w[8];
  int64_t at = -1;  // the position cs, sn were read for
  int kind = -1;    // the stream w was read for
  for (int u = blockIdx.y; u < uq + uk; u += gridDim.y) {
    const bool is_k = u >= uq;
    const Stream& s = is_k ? p.k : p.q;
    if (g.token >= s.tokens) continue;
    const int64_t pos = s.positions ? s.positions[g.token] : g.token % s.period;
    if (kind < 0 || pos != at) load_turn(p, c, g.lane, pos, cs, sn), at = pos;
    if (kind != (is_k ? 1 : 0)) load_weight<T>(s.weight, p.weight_f32, c, w), kind = is_k ? 1 : 0;
    forward_heads<T, LANES>(static_cast<const T*>(s.x) + g.token * s.stride,
                            static_cast<T*>(s.y) + g.token * s.heads * p.D, s.heads, (is_k ? u - uq : u) * kHeads, p, c,
                            w, s.weight != nullptr, cs, sn, g.mask);
  }
}

// The cache write: keys to their page row, queries (if any) to q.y, values
// copied.  Tokens behind the last sequence, at positions below zero or past
// the table, and on pages outside the pool are not written.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) append_kernel(const Params p) {
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place c = place_of(g.lane, p);
  constexpr int kVec = 16 / sizeof(T);
  pdl_wait();
  const int uq = (p.q.heads + kHeads - 1) / kHeads, uk = (p.k.heads + kHeads - 1) / kHeads;
  const int nv = p.k.heads * p.D_v / kVec;  // a token's values in 16-byte words, contiguous on both sides
  const int uv = (nv + LANES * kHeads - 1) / (LANES * kHeads);
  if (g.token >= p.view.tokens) return;
  const int n = seq_of_token<LANES>(p.view, static_cast<int>(g.token), g.mask, g.lane);
  if (n < 0) return;
  const int64_t held = p.view.kv_len[n];
  const int64_t pos = held - (p.view.q_start[n + 1] - g.token);
  const bool in_table = pos >= 0 && pos < (static_cast<int64_t>(p.view.width) << p.view.page_shift);
  const int page = in_table ? page_of(p.view, n, static_cast<int>(pos >> p.view.page_shift)) : -1;
  if (!in_table && g.lane == 0) atomicOr(&g_status_word, kStatusBadIndex);
  const int64_t slot = (static_cast<int64_t>(page) << p.view.page_shift) + (pos & ((1 << p.view.page_shift) - 1));
  float cs[4], sn[4], w[8];
  load_turn(p, c, g.lane, pos, cs, sn);
  int kind = -1;
  for (int u = blockIdx.y; u < uq + uk + uv; u += gridDim.y) {
    if (u >= uq + uk) {
      if (page < 0) continue;
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.x) + g.token * p.v.stride);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.v_pages) + slot * p.k.heads * p.D_v);
      const int i0 = (u - uq - uk) * LANES * kHeads + g.lane;
      uint4 r[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (i0 + i * LANES < nv) r[i] = __ldg(src + i0 + i * LANES);
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (i0 + i * LANES < nv) dst[i0 + i * LANES] = r[i];
      continue;
    }
    const bool is_k = u >= uq;
    if (is_k && page < 0) continue;
    const Stream& s = is_k ? p.k : p.q;
    if (kind != (is_k ? 1 : 0)) load_weight<T>(s.weight, p.weight_f32, c, w), kind = is_k ? 1 : 0;
    T* y = is_k ? static_cast<T*>(p.k_pages) + slot * s.heads * p.D : static_cast<T*>(s.y) + g.token * s.heads * p.D;
    forward_heads<T, LANES>(static_cast<const T*>(s.x) + g.token * s.stride, y, s.heads, (is_k ? u - uq : u) * kHeads, p,
                            c, w, s.weight != nullptr, cs, sn, g.mask);
  }
}

// Backward.  A block walks tokens blockIdx.x, + gridDim.x, ... of its group
// index and all heads, summing dw in registers; the block's sums go to
// partial[block][q, k][D], added by weight_kernel in block order (no atomics:
// the same bits every run).
constexpr int kGradHeads = 2;  // x and dy of two heads in flight

template <typename T, int LANES>
__device__ __forceinline__ void backward_heads(const T* x, const T* dy, T* dx, int heads, int h0, const Params& p,
                                               const Place& c, const float* w, bool norm, const float* cs,
                                               const float* sn, unsigned mask, float* dw) {
  using V = Vec4<T>;
  typename V::type xa[kGradHeads], xb[kGradHeads], ga[kGradHeads], gb[kGradHeads];
#pragma unroll
  for (int i = 0; i < kGradHeads; ++i)
    if (c.live && h0 + i < heads) {
      if (norm) {
        xa[i] = __ldg(reinterpret_cast<const typename V::type*>(x + (h0 + i) * p.D + c.a));
        xb[i] = __ldg(reinterpret_cast<const typename V::type*>(x + (h0 + i) * p.D + c.b));
      }
      ga[i] = __ldg(reinterpret_cast<const typename V::type*>(dy + (h0 + i) * p.D + c.a));
      gb[i] = __ldg(reinterpret_cast<const typename V::type*>(dy + (h0 + i) * p.D + c.b));
    }
#pragma unroll
  for (int i = 0; i < kGradHeads; ++i) {
    if (h0 + i >= heads) break;
    float g[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (c.live) V::unpack(ga[i], g), V::unpack(gb[i], g + 4);
    turn(g, cs, sn, p.interleaved, -1.0f);
    if (norm) {
      float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (c.live) V::unpack(xa[i], f), V::unpack(xb[i], f + 4);
      // both sums at once: mean(g w n) = r * mean(g w x)
      float ss = 0.0f, gx = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss), gx = fmaf(g[e] * w[e], f[e], gx);
      ss = group_sum<LANES>(ss, mask);
      gx = group_sum<LANES>(gx, mask);
      const float d = static_cast<float>(p.D), r = rsqrtf(ss / d + p.eps), m = gx * r / d;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float nrm = f[e] * r;
        dw[e] = fmaf(g[e], nrm, dw[e]);
        g[e] = r * (g[e] * w[e] - nrm * m);
      }
    }
    if (c.live) {
      *reinterpret_cast<typename V::type*>(dx + (h0 + i) * p.D + c.a) = V::pack(g);
      *reinterpret_cast<typename V::type*>(dx + (h0 + i) * p.D + c.b) = V::pack(g + 4);
    }
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Params p) {
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place c = place_of(g.lane, p);
  __shared__ float sums[kThreads / LANES][LANES * 8 + 4];
  pdl_wait();
  constexpr int kGroups = kThreads / LANES;
  for (int is_k = 0; is_k < 2; ++is_k) {
    const Stream& s = is_k ? p.k : p.q;
    float w[8], dw[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    load_weight<T>(s.weight, p.weight_f32, c, w);
    // grid.y shares the heads; without a norm nothing is summed
    for (int64_t t = g.token; t < s.tokens; t += static_cast<int64_t>(gridDim.x) * kGroups) {
      float cs[4], sn[4];
      load_turn(p, c, g.lane, s.positions ? s.positions[t] : t % s.period, cs, sn);
      for (int h = 0; h < s.heads; h += kGradHeads)
        backward_heads<T, LANES>(static_cast<const T*>(s.x) + t * s.stride, static_cast<const T*>(s.dy) + t * s.dy_stride,
                                 static_cast<T*>(s.y) + t * s.heads * p.D, s.heads, h, p, c, w, s.weight != nullptr, cs,
                                 sn, g.mask, dw);
    }
    if (!s.weight) continue;  // the same for the whole grid
    const int row = threadIdx.x / LANES;
    __syncthreads();
    if (c.live) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[row][c.a + e] = dw[e], sums[row][c.b + e] = dw[4 + e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += kThreads) {
      float a = 0.0f;
#pragma unroll
      for (int r = 0; r < kGroups; ++r) a += sums[r][i];
      p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + is_k) * p.D + i] = a;
    }
  }
}

// dw[i] = sum over blocks of partial[block][stream][i]: one block of 32 x 32
// threads for 32 features of one stream (blockIdx.y).
template <typename T>
__global__ void __launch_bounds__(1024) weight_kernel(const Params p) {
  __shared__ float part[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, i = blockIdx.x * 32 + x;
  void* dst = blockIdx.y ? p.dw_k : p.dw_q;
  if (!dst) return;
  float a = 0.0f;
  if (i < p.D)
    for (int b = y; b < p.blocks; b += 32) a += p.partial[(static_cast<int64_t>(b) * 2 + blockIdx.y) * p.D + i];
  part[y][x] = a;
  __syncthreads();
  if (y == 0 && i < p.D) {
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) s += part[r][x];
    if (p.weight_f32)
      static_cast<float*>(dst)[i] = s;
    else
      static_cast<T*>(dst)[i] = from_f<T>(s);
  }
}

}  // namespace rotary
}  // namespace sdpa_b200
