// Query/key head norms with the position rotation, and the write of new keys
// and values into the paged cache, which applies them on the way.
//
//   n = x * rsqrt(mean(x^2) + eps)           (per head; skipped without a weight)
//   y = R(pos) (n * w)                       R turns feature pairs by pos * base^(-2i/rot)
// Backward: g = R(pos)^T dy,  dw = sum g * n,  dx = rsqrt(..) * (g w - n * mean(g w n)).
//
// Bound: HBM bytes (forward: x in, y out; backward: x, dy in, dx out); per
// element about ten fp32 operations, so the work beside the loads is kept short:
// a group of LANES lanes owns one head row, eight features a lane, so the row's
// sum is three or four shuffles; both members of every rotated pair sit in one
// lane (for pairs (i, i + rot/2) features 4j.. and rot/2 + 4j.., for neighbouring
// pairs 8j..), weights, cosines and sines are multiplied once a token, and the
// products go in packed pairs (f32x2).  A group walks the heads of one token,
// four at a time with all their loads ahead of the arithmetic.  32768 tokens x
// 32 heads x 128 in fp16: forward 99 us (537 MB, 5.4 TB/s); backward of 40 heads 183 us
// (1007 MB, 5.5 TB/s).  Measured worse: the weights and the turn applied apart (120 us forward);
// sixteen features a lane, with 16-byte loads and fewer instructions but over 110
// registers (118 us); the forward's loads through a ring as the backward's (99 us).
// All arithmetic is fp32, rounded to T once, at the store.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace sdpa_b200 {
namespace rotary {

constexpr int kThreads = 256;
constexpr int E = 4;              // features of one of a lane's two runs
constexpr int kGradBlocks = 592;  // most blocks of the backward (rows of its workspace)

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
  float eps, inv_D;    // inv_D = 1 / D
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

// E consecutive features as loaded, and as floats.
template <typename T>
struct Raw {
  uint32_t w[E * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) {
    if (sizeof(w) == 8) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if (sizeof(w) == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(w) / 16); ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 4); ++i) {
      if (sizeof(T) == 2) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = x.x, f[2 * i + 1] = x.y;
      } else {
        f[i] = __uint_as_float(w[i]);
      }
    }
  }
  __device__ __forceinline__ void pack(const float* f) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 4); ++i)
      w[i] = sizeof(T) == 2 ? pack_half2(f[2 * i], f[2 * i + 1]) : __float_as_uint(f[i]);
  }
};

// Where a lane's features lie, two runs of E, and whether they turn.
template <bool INTER>
struct Place {
  int a, b;           // first feature of each run
  int angle;          // of its E pairs: index of the first
  bool live, turned;  // inside the row; inside the rotated part
  __device__ __forceinline__ Place(int lane, const Params& p) {
    live = lane * 2 * E < p.D;
    turned = p.table && lane * 2 * E < p.rot;
    const bool halves = turned && !INTER;
    a = halves ? lane * E : lane * 2 * E;
    b = halves ? p.rot / 2 + lane * E : lane * 2 * E + E;
    angle = lane * E;
  }
  // registers of pair e's members
  static __device__ __forceinline__ constexpr int first(int e) { return INTER ? 2 * e : e; }
  static __device__ __forceinline__ constexpr int second(int e) { return INTER ? 2 * e + 1 : E + e; }
};

template <typename T, bool INTER>
__device__ __forceinline__ void load_weight(const void* w, int f32, const Place<INTER>& c, float* out) {
#pragma unroll
  for (int e = 0; e < 2 * E; ++e) out[e] = 1.0f;
  if (!w || !c.live) return;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    out[e] = f32 ? static_cast<const float*>(w)[c.a + e] : to_f<T>(static_cast<const T*>(w)[c.a + e]);
    out[E + e] = f32 ? static_cast<const float*>(w)[c.b + e] : to_f<T>(static_cast<const T*>(w)[c.b + e]);
  }
}

// Cosines and sines of a lane's E pairs at `pos` (1 and 0 where nothing turns).
template <bool INTER>
__device__ __forceinline__ void load_turn(const Params& p, const Place<INTER>& c, int lane, int64_t pos, float* cs,
                                          float* sn) {
#pragma unroll
  for (int e = 0; e < E; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
  if (!p.table) return;
  if (pos < 0 || pos >= p.max_positions) {
    if (lane == 0) atomicOr(&g_status_word, kStatusBadIndex);
    pos = pos < 0 ? 0 : p.max_positions - 1;
  }
  if (c.turned) {
    const float* row = p.table + pos * p.rot + c.angle;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + e));
      cs[e] = a.x, cs[e + 1] = a.y, cs[e + 2] = a.z, cs[e + 3] = a.w;
    }
    const float* srow = row + p.rot / 2;  // (a multiple of four floats)
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 b = __ldg(reinterpret_cast<const float4*>(srow + e));
      sn[e] = b.x, sn[e + 1] = b.y, sn[e + 2] = b.z, sn[e + 3] = b.w;
    }
  }
}

// The turn of weighted features, y = R (x w): first = x1 ca - x2 sb, second = x2 cb + x1 sa.
struct Turn {
  float ca[E], sb[E], cb[E], sa[E];
  template <bool INTER>
  __device__ __forceinline__ void set(const float* w, const float* cs, const float* sn) {
    using P = Place<INTER>;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      ca[e] = w[P::first(e)] * cs[e];
      sa[e] = w[P::first(e)] * sn[e];
      cb[e] = w[P::second(e)] * cs[e];
      sb[e] = -w[P::second(e)] * sn[e];
    }
  }
};

template <int LANES>
__device__ __forceinline__ float group_sum(float x, unsigned mask) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d >>= 1) x += __shfl_xor_sync(mask, x, d);
  return x;
}

// Norm, rotation and store of heads [h0, h0 + N) of one token, as loaded.
template <typename T, int LANES, bool INTER, int N>
__device__ __forceinline__ void forward_heads(const Raw<T>* ra, const Raw<T>* rb, T* y, int heads, int h0, const Params& p,
                                              const Place<INTER>& c, const Turn& w, bool norm, unsigned mask) {
  using P = Place<INTER>;
  T *ya = y + h0 * p.D + c.a, *yb = y + h0 * p.D + c.b;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (h0 + i >= heads) break;  // the same for every lane of the group
    float f[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) f[e] = 0.0f;
    if (c.live) ra[i].unpack(f), rb[i].unpack(f + E);
    float r = 1.0f;
    if (norm) {
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * E; e += 2) ffma2(s0, s1, f[e], f[e + 1], f[e], f[e + 1], s0, s1);
      r = rsqrtf(group_sum<LANES>(s0 + s1, mask) * p.inv_D + p.eps);
    }
    float z[2 * E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float u0, u1, v0, v1;
      const float a0 = f[P::first(e)], a1 = f[P::first(e + 1)], b0 = f[P::second(e)], b1 = f[P::second(e + 1)];
      fmul2(u0, u1, a0, a1, w.ca[e], w.ca[e + 1]);
      ffma2(u0, u1, b0, b1, w.sb[e], w.sb[e + 1], u0, u1);
      fmul2(v0, v1, b0, b1, w.cb[e], w.cb[e + 1]);
      ffma2(v0, v1, a0, a1, w.sa[e], w.sa[e + 1], v0, v1);
      fmul2(z[P::first(e)], z[P::first(e + 1)], u0, u1, r, r);
      fmul2(z[P::second(e)], z[P::second(e + 1)], v0, v1, r, r);
    }
    if (c.live) {
      Raw<T> o;
      o.pack(z);
      o.store(ya + i * p.D);
      o.pack(z + E);
      o.store(yb + i * p.D);
    }
  }
}

// A lane's ring in shared memory: words of one run of E features, kThreads
// apart, written by the lane's own cp.async and read by itself (no barrier).
template <typename T>
struct Ring {
  static constexpr int kWord = E * sizeof(T);  // 8 or 16 bytes
  uint8_t* base;
  __device__ __forceinline__ explicit Ring(uint8_t* smem) : base(smem + threadIdx.x * kWord) {}
  __device__ __forceinline__ void copy(int word, const T* src) {
    const uint32_t dst = smem_u32(base + word * (kThreads * kWord));
    if (kWord == 8)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
    else
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  }
  __device__ __forceinline__ Raw<T> read(int word) const {
    Raw<T> r;
    if (kWord == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(base + word * (kThreads * kWord));
      r.w[0] = x.x, r.w[1] = x.y;
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(base + word * (kThreads * kWord));
      r.w[0] = x.x, r.w[1] = x.y, r.w[kWord / 4 - 2] = x.z, r.w[kWord / 4 - 1] = x.w;
    }
    return r;
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  template <int N>
  static __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  }
};

constexpr int kHeadsAhead = 4;  // heads a group takes at a time
// Stages of the backward's ring, each x and dy of two heads: eight words a lane.
template <typename T>
constexpr int kStages = sizeof(T) == 2 ? 4 : 2;
template <typename T>
constexpr int kStageBytes = 8 * kThreads * E * static_cast<int>(sizeof(T));
// Blocks an SM (fp32 holds twice the loads): forward (fp16: 64 registers a
// thread, 44 bytes of them spilled), and append, whose addresses take more (fp16:
// 80 registers and 64 bytes spilled; 5251 tokens x 48 heads x 128: 35 us against 37
// with four blocks, 46 with two).
template <typename T>
constexpr int kBlocks = sizeof(T) == 2 ? 4 : 3;
template <typename T>
constexpr int kAppendBlocks = sizeof(T) == 2 ? 3 : 2;
// Head groups of a stream.
__host__ __device__ __forceinline__ int units_of(int heads, int ahead) { return (heads + ahead - 1) / ahead; }

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
template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads, kBlocks<T>) forward_kernel(const Params p) {
  constexpr int N = kHeadsAhead;
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place<INTER> c(g.lane, p);
  pdl_wait();
  const int uq = units_of(p.q.heads, N), uk = units_of(p.k.heads, N);
  const int64_t tokens = max(p.q.tokens, p.k.tokens);
  if (g.token >= tokens) return;
  Turn turn;
  int64_t at = -1;  // the position and stream that `turn` is of
  int kind = -1;
  for (int u = blockIdx.y; u < uq + uk; u += gridDim.y) {
    const bool is_k = u >= uq;
    const Stream& s = is_k ? p.k : p.q;
    if (g.token >= s.tokens) continue;
    const int h0 = (is_k ? u - uq : u) * N;
    const T* x = static_cast<const T*>(s.x) + g.token * s.stride + h0 * p.D;
    Raw<T> ra[N], rb[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c.live && h0 + i < s.heads) ra[i].load(x + i * p.D + c.a), rb[i].load(x + i * p.D + c.b);
    const int64_t pos = s.positions ? s.positions[g.token] : static_cast<int>(g.token) % s.period;
    if (kind != (is_k ? 1 : 0) || pos != at) {
      float cs[E], sn[E], w[2 * E];
      load_turn(p, c, g.lane, pos, cs, sn);
      load_weight<T>(s.weight, p.weight_f32, c, w);
      turn.set<INTER>(w, cs, sn);
      kind = is_k ? 1 : 0;
      at = pos;
    }
    forward_heads<T, LANES, INTER, N>(ra, rb, static_cast<T*>(s.y) + g.token * s.heads * p.D, s.heads, h0, p, c, turn,
                                      s.weight != nullptr, g.mask);
  }
}

// The cache write: keys to their page row, queries (if any) to q.y, values
// copied.  Tokens behind the last sequence, at positions below zero or past
// the table, and on pages outside the pool are not written.
constexpr int kCopyWords = 4;  // 16-byte words of the values a lane has in flight
template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads, kAppendBlocks<T>) append_kernel(const Params p) {
  constexpr int N = kHeadsAhead;
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place<INTER> c(g.lane, p);
  constexpr int kVec = 16 / sizeof(T);
  pdl_wait();
  const int uq = units_of(p.q.heads, N), uk = units_of(p.k.heads, N);
  const int nv = p.k.heads * p.D_v / kVec;  // a token's values in 16-byte words, contiguous on both sides
  const int uv = units_of(nv, LANES * kCopyWords), units = uq + uk + uv;
  if (g.token >= p.view.tokens) return;
  Raw<T> ra[N], rb[N];
  uint4 words[kCopyWords];
  auto load = [&](int u) {
    if (u >= uq + uk) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.x) + g.token * p.v.stride);
      const int i0 = (u - uq - uk) * LANES * kCopyWords + g.lane;
#pragma unroll
      for (int i = 0; i < kCopyWords; ++i)
        if (i0 + i * LANES < nv) words[i] = __ldg(src + i0 + i * LANES);
    } else {
      const Stream& s = u >= uq ? p.k : p.q;
      const int h0 = (u >= uq ? u - uq : u) * N;
      const T* x = static_cast<const T*>(s.x) + g.token * s.stride + h0 * p.D;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c.live && h0 + i < s.heads) ra[i].load(x + i * p.D + c.a), rb[i].load(x + i * p.D + c.b);
    }
  };
  int u = blockIdx.y;
  load(u);  // on its way while the token's place is looked up (four dependent reads)
  if (blockIdx.x == 0 && blockIdx.y == 0) starts_check(p.view, min(static_cast<int64_t>(kThreads), p.view.tokens * int64_t(LANES)));
  const int n = seq_of_token<LANES>(p.view, static_cast<int>(g.token), g.mask, g.lane);
  if (n < 0) return;
  const int64_t held = p.view.kv_len[n];
  const int64_t end = min(p.view.q_start[n + 1], p.view.tokens);
  if (p.view.q_start[n] > g.token || g.token >= end) return;  // (starts that descend)
  const int64_t pos = held - (end - g.token);
  const bool in_table = pos >= 0 && pos < (static_cast<int64_t>(p.view.width) << p.view.page_shift);
  const int page = in_table ? page_of(p.view, n, static_cast<int>(pos >> p.view.page_shift)) : -1;
  if (!in_table && g.lane == 0) atomicOr(&g_status_word, kStatusBadIndex);
  const int64_t slot = (static_cast<int64_t>(page) << p.view.page_shift) + (pos & ((1 << p.view.page_shift) - 1));
  float cs[E], sn[E];
  load_turn(p, c, g.lane, pos, cs, sn);
  Turn turn;
  int kind = -1;  // the stream that `turn` is of
  while (true) {
    if (u >= uq + uk) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.v_pages) + slot * p.k.heads * p.D_v);
      const int i0 = (u - uq - uk) * LANES * kCopyWords + g.lane;
#pragma unroll
      for (int i = 0; i < kCopyWords; ++i)
        if (page >= 0 && i0 + i * LANES < nv) dst[i0 + i * LANES] = words[i];
    } else {
      const bool is_k = u >= uq;
      const Stream& s = is_k ? p.k : p.q;
      if (!is_k || page >= 0) {
        if (kind != (is_k ? 1 : 0)) {
          float w[2 * E];
          load_weight<T>(s.weight, p.weight_f32, c, w);
          turn.set<INTER>(w, cs, sn);
          kind = is_k ? 1 : 0;
        }
        T* y = is_k ? static_cast<T*>(p.k_pages) + slot * s.heads * p.D : static_cast<T*>(s.y) + g.token * s.heads * p.D;
        forward_heads<T, LANES, INTER, N>(ra, rb, y, s.heads, (is_k ? u - uq : u) * N, p, c, turn, s.weight != nullptr,
                                          g.mask);
      }
    }
    if ((u += gridDim.y) >= units) break;
    load(u);
  }
}

// Backward of heads [h0, h0 + N) of one token, as loaded (x: a, b, dy: a, b of
// each head): dx, and dw summed.
template <typename T, int LANES, bool INTER, int N>
__device__ __forceinline__ void backward_heads(const Raw<T> (&in)[N][4], T* dx, int heads, int h0, const Params& p,
                                               const Place<INTER>& c, const float* w, bool norm, const float* cs,
                                               const float* sn, unsigned mask, float* dw) {
  using P = Place<INTER>;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (h0 + i >= heads) break;
    float d[2 * E], g[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) d[e] = 0.0f;
    if (c.live) in[i][2].unpack(d), in[i][3].unpack(d + E);
#pragma unroll
    for (int e = 0; e < E; e += 2) {  // g = R^T dy
      const float a0 = d[P::first(e)], a1 = d[P::first(e + 1)], b0 = d[P::second(e)], b1 = d[P::second(e + 1)];
      float u0, u1, v0, v1;
      fmul2(u0, u1, a0, a1, cs[e], cs[e + 1]);
      ffma2(g[P::first(e)], g[P::first(e + 1)], b0, b1, sn[e], sn[e + 1], u0, u1);
      fmul2(v0, v1, b0, b1, cs[e], cs[e + 1]);
      ffma2(g[P::second(e)], g[P::second(e + 1)], a0, a1, -sn[e], -sn[e + 1], v0, v1);
    }
    if (norm) {
      float f[2 * E], gw[2 * E];
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) f[e] = 0.0f;
      if (c.live) in[i][0].unpack(f), in[i][1].unpack(f + E);
      // both sums at once: mean(g w n) = r * mean(g w x)
      float s0 = 0.0f, s1 = 0.0f, t0 = 0.0f, t1 = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * E; e += 2) {
        ffma2(s0, s1, f[e], f[e + 1], f[e], f[e + 1], s0, s1);
        fmul2(gw[e], gw[e + 1], g[e], g[e + 1], w[e], w[e + 1]);
        ffma2(t0, t1, gw[e], gw[e + 1], f[e], f[e + 1], t0, t1);
      }
      const float ss = group_sum<LANES>(s0 + s1, mask), gx = group_sum<LANES>(t0 + t1, mask);
      const float r = rsqrtf(ss * p.inv_D + p.eps), m = -gx * r * p.inv_D;
#pragma unroll
      for (int e = 0; e < 2 * E; e += 2) {
        float n0, n1, u0, u1;
        fmul2(n0, n1, f[e], f[e + 1], r, r);
        ffma2(dw[e], dw[e + 1], g[e], g[e + 1], n0, n1, dw[e], dw[e + 1]);
        ffma2(u0, u1, n0, n1, m, m, gw[e], gw[e + 1]);
        fmul2(g[e], g[e + 1], u0, u1, r, r);
      }
    }
    if (c.live) {
      Raw<T> o;
      o.pack(g);
      o.store(dx + (h0 + i) * p.D + c.a);
      o.pack(g + E);
      o.store(dx + (h0 + i) * p.D + c.b);
    }
  }
}

// A block walks tokens blockIdx.x, + gridDim.x, .. (grid.y: shares of the heads
// when there are few tokens), summing dw in registers; its sums go to
// partial[block][q, k][D], added by weight_kernel in block order (no atomics: the
// same bits every run).  The loads run kStages - 1 head pairs ahead, through
// shared memory: at its registers two blocks an SM fit, whose own loads are too few
// in flight (8192 tokens x 40 heads x 128 fp16: 61 us against 75 without the ring, 4099 x 32 x 64
// fp32, two head pairs a group: 25 and 27).
template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const Params p) {
  constexpr int N = 2, ST = kStages<T>;  // x and dy of two heads a stage
  constexpr int kGroups = kThreads / LANES;
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_launch_dependents();
  const Group<LANES> g;
  const Place<INTER> c(g.lane, p);
  Ring<T> ring(smem);
  __shared__ float sums[kGroups][LANES * 2 * E + 4];
  pdl_wait();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  for (int is_k = 0; is_k < 2; ++is_k) {
    const Stream& s = is_k ? p.k : p.q;
    const bool norm = s.weight != nullptr;
    float w[2 * E], dw[2 * E];
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) dw[e] = 0.0f;
    load_weight<T>(s.weight, p.weight_f32, c, w);
    int64_t t_in = g.token;  // the walk of the loads
    int h_in = blockIdx.y * N, stage_in = 0, stage = 0;
    auto load = [&]() {
      if (t_in < s.tokens && h_in < s.heads) {
        if (c.live) {
          const T* x = static_cast<const T*>(s.x) + t_in * s.stride + h_in * p.D;
          const T* dy = static_cast<const T*>(s.dy) + t_in * s.dy_stride + h_in * p.D;
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (h_in + i < s.heads) {
              const int word = (stage_in * N + i) * 4;
              if (norm) ring.copy(word, x + i * p.D + c.a), ring.copy(word + 1, x + i * p.D + c.b);
              ring.copy(word + 2, dy + i * p.D + c.a), ring.copy(word + 3, dy + i * p.D + c.b);
            }
        }
        if ((h_in += gridDim.y * N) >= s.heads) h_in = blockIdx.y * N, t_in += step;
        if (++stage_in == ST) stage_in = 0;
      }
      ring.commit();
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) load();
    for (int64_t t = g.token; t < s.tokens; t += step) {
      float cs[E], sn[E];
      load_turn(p, c, g.lane, s.positions ? s.positions[t] : static_cast<int>(t) % s.period, cs, sn);
      for (int h = blockIdx.y * N; h < s.heads; h += gridDim.y * N) {
        Raw<T> in[N][4];
        ring.template wait<ST - 2>();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) in[i][k] = ring.read((stage * N + i) * 4 + k);
        if (++stage == ST) stage = 0;
        load();  // into the stage that the last pair has left
        backward_heads<T, LANES, INTER, N>(in, static_cast<T*>(s.y) + t * s.heads * p.D, s.heads, h, p, c, w, norm, cs, sn,
                                           g.mask, dw);
      }
    }
    if (!s.weight) continue;  // the same for the whole grid
    const int row = threadIdx.x / LANES;
    __syncthreads();
    if (c.live) {
#pragma unroll
      for (int e = 0; e < E; ++e) sums[row][c.a + e] = dw[e], sums[row][c.b + e] = dw[E + e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += kThreads) {
      float a = 0.0f;
#pragma unroll 8
      for (int r = 0; r < kGroups; ++r) a += sums[r][i];
      p.partial[((static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * 2 + is_k) * p.D + i] = a;
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
