// Attention of new tokens over the paged cache, for sequences with few of
// them (single tokens, drafted ones), fp16 and fp32.
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j,   stats_i = max + ln(sum + 1e-6)
//
// Bound: the bytes of the K and V rows held, read once (each serves only the
// rows of its head group).  The G = H_q / H_kv query heads of a KV head and the
// sequence's new tokens are packed into rows r = token * G + g, 16 to a tile,
// so all of them share one reading.  The products go through warp-level
// matrix instructions (m16n8k16 fp16; m16n8k8 tf32 three times a product for
// fp32): 16 rows are a tenth of a tcgen05 tile, and its operands would have to
// pass through shared memory and TMEM, while these take them from registers.
//
// Register operands straight from global memory: a matrix product may take its
// inner index in any order as long as both operands agree.  A lane (g = lane/4,
// t = lane%4) therefore reads 16-byte words, K[key g][32i + 8t ..], and uses
// their four 32-bit parts as the B operands of two instructions, with Q's A
// operands laid out the same way; V[key 2t][64i + 8g ..] likewise, neighbouring
// keys joined by byte permutes.  No shared memory, no barrier in the loop, and
// every warp streams on its own: block of kKeys keys = K and V words of one
// block in flight while the previous is computed.
//
// Work: every (sequence, KV head, row tile) item has ceil(held / 64) tiles of
// 64 keys; the tiles of all items, in order, are cut into equal ranges, one per
// CTA, so long and short sequences load the device evenly.  An item that lies
// in one CTA is finished there; one that is cut leaves partial sums (at most two
// a CTA) that merge_kernel joins.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace sdpa_b200 {
namespace paged {

constexpr int kTile = 64;       // keys of one unit of work
constexpr int kRows = 16;       // packed query rows of one matrix tile
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct Params {
  const void* q;
  const void* k_pages;
  const void* v_pages;
  void* out;              // [tokens, H_q, D_v]
  float* stats;           // [tokens, H_q]
  int64_t q_stride;       // elements between tokens of q
  PagedView view;
  int H_q, H_kv, G, D, D_v;
  float scale_log2;
  int causal;
  // workspace
  float* part_o;          // [ctas, 2, rows, DB] unnormalised sums
  float2* part_ml;        // [ctas, 2, rows] (max, sum), log2 units
  int4* part_item;        // [ctas] (sequence, head, row tile, CTAs after this one that hold the rest; -1: none)
  int sms;                // SMs of the device
  uint64_t timeout_ns;
};

__device__ __forceinline__ void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_1688(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, both tf32 values: hi is x rounded to 11 bits (half away from
// zero, by an integer add: the conversion instruction runs at a fraction of
// the rate), lo the rounded rest.
__device__ __forceinline__ void split_fast(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}

// Per type: keys of a warp's block and 16-byte words of one row.
template <typename T>
struct Kind;
template <>
struct Kind<__half> {
  static constexpr int kKeys = 16;
};
template <>
struct Kind<float> {
  static constexpr int kKeys = 8;
};

// 16 bytes of a read-only row, kept out of L1 unless several warps of the CTA
// read the same rows.
template <bool SHARED_ROWS>
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 r;
  if (SHARED_ROWS)
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
  return r;
}

__device__ __forceinline__ int row_tiles(const Params& p, const SeqLens& s, int rows) {
  return static_cast<int>((static_cast<int64_t>(s.count) * p.G + rows - 1) / rows);
}
__device__ __forceinline__ int key_tiles(const SeqLens& s) { return s.held > 0 ? (s.held + kTile - 1) / kTile : 1; }
// Tiles of all items of sequence n.
__device__ __forceinline__ int64_t seq_work(const Params& p, int n, int rows) {
  const SeqLens s = seq_lens(p.view, n);
  return static_cast<int64_t>(row_tiles(p, s, rows)) * p.H_kv * key_tiles(s);
}

template <int DB, int MT>
struct Smem {
  static constexpr int kOStride = DB + 4;
  float o[kWarps][kRows][kOStride];
  float m[kWarps][kRows], l[kWarps][kRows];
};

// Four columns of one output row from its sums (and, at column 0, its stats):
// the op's row rule, stats = max + ln(l + 1e-6), rows that saw no key are zero.
template <typename T>
__device__ __forceinline__ void store_row(const Params& p, int64_t row, int c, const float4& acc, float m, float l) {
  const float inv = l > kEps ? 1.0f / l : 0.0f;
  if (c == 0) p.stats[row] = (m == -INFINITY ? kNegInit : m * kLn2) + logf(l + kEps);
  if (c >= p.D_v) return;
  T* dst = static_cast<T*>(p.out) + row * p.D_v + c;
  if (sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  } else {
    *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
}

// MT row tiles of 16 by 4 / MT shares of the keys: with more than one row tile
// the warps of a share read the same rows (the second reading hits L1).
template <typename T, int DB, int MT>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const Params p) {
  constexpr int KS = kWarps / MT;
  constexpr int KEYS = Kind<T>::kKeys;
  constexpr bool HALF = sizeof(T) == 2;
  constexpr int KW = HALF ? DB / 32 : DB / 16;        // K words a lane reads of one key
  constexpr int KN = KEYS / 8;                        // keys a lane reads K of
  constexpr int VW = HALF ? DB / 64 : DB / 32;        // V words a lane reads of one key
  constexpr int VN = HALF ? 4 : 2;                    // keys a lane reads V of
  constexpr int NO = DB / 8;                          // output column tiles
  constexpr int ROWS = kRows * MT;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem<DB, MT>& sm = *reinterpret_cast<Smem<DB, MT>*>(smem_raw);
  // fp32: Q's operands, hi and lo, as [row tile][word][4][lane] float4
  uint4* const sq = reinterpret_cast<uint4*>(smem_raw + sizeof(Smem<DB, MT>));
  __shared__ int64_t s_sum[kWarps];
  __shared__ int64_t s_base;
  __shared__ int s_seq;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mt = warp % MT, ks = warp / MT;
  const int g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's range of tiles
  const int per = (p.view.seqs + kThreads - 1) / kThreads;
  int64_t mine = 0;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < p.view.seqs) mine += seq_work(p, tid * per + i, ROWS);
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
  if (tid == 0) p.part_item[blockIdx.x] = make_int4(0, 0, 0, -1);
  if (blockIdx.x >= ctas) return;
  const int64_t w0 = total * blockIdx.x / ctas, w1 = total * (blockIdx.x + 1) / ctas;
  const int64_t excl = before + incl - mine;
  if (excl <= w0 && w0 < excl + mine) {
    int64_t base = excl;
    int n = tid * per;
    for (;; ++n) {
      const int64_t s = seq_work(p, n, ROWS);
      if (w0 < base + s) break;
      base += s;
    }
    s_seq = n;
    s_base = base;
  }
  __syncthreads();
  int n = s_seq;
  int64_t base = s_base;

  const int64_t k_row = static_cast<int64_t>(p.H_kv) * p.D, v_row = static_cast<int64_t>(p.H_kv) * p.D_v;
  const int page_shift = p.view.page_shift, page_mask = (1 << page_shift) - 1;
  const bool whole = p.D == DB && p.D_v == DB;

  for (int64_t w = w0; w < w1;) {
    const SeqLens sl = seq_lens(p.view, n);
    const int rt = row_tiles(p, sl, ROWS), nt = key_tiles(sl);
    const int64_t work = static_cast<int64_t>(rt) * p.H_kv * nt;
    if (w >= base + work) {
      base += work;
      ++n;
      continue;
    }
    const int64_t local = w - base;
    const int64_t item = local / nt;
    const int tile0 = static_cast<int>(local - item * nt);
    const int head = static_cast<int>(item / rt), rtile = static_cast<int>(item - static_cast<int64_t>(head) * rt);
    const int tiles = static_cast<int>(min(static_cast<int64_t>(nt - tile0), w1 - w));

    // ---- rows of this warp
    const int total_rows = sl.count * p.G;
    const int r0 = (rtile * MT + mt) * kRows;
    const int ra = r0 + g, rb = r0 + g + 8;
    const bool va = ra < total_rows, vb = rb < total_rows;
    const int shift = sl.held - sl.count;  // position of the first new token
    // keys a row sees: [0, lim)
    const int lim_a = p.causal ? min(sl.held, shift + ra / p.G + 1) : sl.held;
    const int lim_b = p.causal ? min(sl.held, shift + rb / p.G + 1) : sl.held;
    const int lim_0 = p.causal ? min(sl.held, shift + r0 / p.G + 1) : sl.held;  // the least of the warp's
    const T* qa = static_cast<const T*>(p.q) + (sl.begin + ra / p.G) * p.q_stride + (head * p.G + ra % p.G) * p.D;
    const T* qb = static_cast<const T*>(p.q) + (sl.begin + rb / p.G) * p.q_stride + (head * p.G + rb % p.G) * p.D;
    uint4 qf[HALF ? 2 * KW : 1];
    if (HALF) {
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        const int d = 32 * i + 8 * t;
        qf[2 * i] = va && d < p.D ? ldg16<true>(qa + d) : make_uint4(0, 0, 0, 0);
        qf[2 * i + 1] = vb && d < p.D ? ldg16<true>(qb + d) : make_uint4(0, 0, 0, 0);
      }
    } else {
      __syncthreads();  // the previous item's readers are done
      if (ks == 0) {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const int d = 16 * i + 4 * t;
          const uint4 a = va && d < p.D ? ldg16<true>(qa + d) : make_uint4(0, 0, 0, 0);
          const uint4 b = vb && d < p.D ? ldg16<true>(qb + d) : make_uint4(0, 0, 0, 0);
          uint4 ah, al, bh, bl;
          split_fast(__uint_as_float(a.x), ah.x, al.x), split_fast(__uint_as_float(a.y), ah.y, al.y);
          split_fast(__uint_as_float(a.z), ah.z, al.z), split_fast(__uint_as_float(a.w), ah.w, al.w);
          split_fast(__uint_as_float(b.x), bh.x, bl.x), split_fast(__uint_as_float(b.y), bh.y, bl.y);
          split_fast(__uint_as_float(b.z), bh.z, bl.z), split_fast(__uint_as_float(b.w), bh.w, bl.w);
          // the operand order of the instruction: (row g, k t) (row g+8, k t) (row g, k t+4) (row g+8, k t+4)
          uint4* dst = sq + ((mt * KW + i) * 4) * 32 + lane;
          dst[0] = make_uint4(ah.x, bh.x, ah.y, bh.y);
          dst[32] = make_uint4(ah.z, bh.z, ah.w, bh.w);
          dst[64] = make_uint4(al.x, bl.x, al.y, bl.y);
          dst[96] = make_uint4(al.z, bl.z, al.w, bl.w);
        }
      }
      __syncthreads();
    }

    // ---- the warp's blocks of keys
    const int blk0 = tile0 * (kTile / KEYS) + ks;
    const int blk1 = (min((tile0 + tiles) * kTile, sl.held) + KEYS - 1) / KEYS;
    float o[NO][4];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;
    uint4 kf[KN][KW], vf[VN][VW];
    const T* const kp = static_cast<const T*>(p.k_pages) + static_cast<int64_t>(head) * p.D;
    const T* const vp = static_cast<const T*>(p.v_pages) + static_cast<int64_t>(head) * p.D_v;

    // pages of the next 32 blocks, one a lane, read a batch ahead
    auto pages_from = [&](int blk) {
      const int key = (blk + lane * KS) * KEYS;
      return key < sl.held && blk + lane * KS < blk1 ? page_of(p.view, n, key >> page_shift) : -1;
    };
    auto load_k = [&](int blk, int page) {
      const int key = blk * KEYS;
      const T* row = kp + ((static_cast<int64_t>(page) << page_shift) + (key & page_mask)) * k_row;
      if (whole && page >= 0 && key + KEYS <= sl.held) {
#pragma unroll
        for (int a = 0; a < KN; ++a)
#pragma unroll
          for (int i = 0; i < KW; ++i)
            kf[a][i] = ldg16<(MT > 1)>(row + (8 * a + g) * k_row + (HALF ? 32 * i + 8 * t : 16 * i + 4 * t));
      } else {
#pragma unroll
        for (int a = 0; a < KN; ++a)
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            const int d = HALF ? 32 * i + 8 * t : 16 * i + 4 * t;
            kf[a][i] = make_uint4(0, 0, 0, 0);
            if (page >= 0 && key + 8 * a + g < sl.held && d < p.D) kf[a][i] = ldg16<(MT > 1)>(row + (8 * a + g) * k_row + d);
          }
      }
    };
    auto load_v = [&](int blk, int page) {
      const int key = blk * KEYS;
      const T* row = vp + ((static_cast<int64_t>(page) << page_shift) + (key & page_mask)) * v_row;
      if (whole && page >= 0 && key + KEYS <= sl.held) {
#pragma unroll
        for (int a = 0; a < VN; ++a)
#pragma unroll
          for (int i = 0; i < VW; ++i)
            vf[a][i] = ldg16<(MT > 1)>(row + (8 * (a >> 1) + 2 * t + (a & 1)) * v_row + (HALF ? 64 * i + 8 * g : 32 * i + 4 * g));
      } else {  // rows behind the sequence read as zeros: whatever the pool holds there stays out of the sums
#pragma unroll
        for (int a = 0; a < VN; ++a)
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            const int d = HALF ? 64 * i + 8 * g : 32 * i + 4 * g, r = 8 * (a >> 1) + 2 * t + (a & 1);
            vf[a][i] = make_uint4(0, 0, 0, 0);
            if (page >= 0 && key + r < sl.held && d < p.D_v) vf[a][i] = ldg16<(MT > 1)>(row + r * v_row + d);
          }
      }
    };

    int pages = pages_from(blk0), pages_next = pages_from(blk0 + 32 * KS);
    int page = __shfl_sync(0xffffffffu, pages, 0);
    if (blk0 < blk1) load_k(blk0, page), load_v(blk0, page);
    int it = 0;
    for (int blk = blk0; blk < blk1; blk += KS) {
      ++it;
      if ((it & 31) == 0) {
        pages = pages_next;
        pages_next = pages_from(blk + KS + 32 * KS);
      }
      const int page_n = __shfl_sync(0xffffffffu, pages, it & 31);
      const bool more = blk + KS < blk1;
      const int key0 = blk * KEYS;
      // S = Q K^T
      float s[KN][4];
#pragma unroll
      for (int a = 0; a < KN; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] = 0.0f;
      if (HALF) {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t a0[4] = {qf[2 * i].x, qf[2 * i + 1].x, qf[2 * i].y, qf[2 * i + 1].y};
          const uint32_t a1[4] = {qf[2 * i].z, qf[2 * i + 1].z, qf[2 * i].w, qf[2 * i + 1].w};
#pragma unroll
          for (int a = 0; a < KN; ++a) {
            mma_16816(s[a], a0, kf[a][i].x, kf[a][i].y);
            mma_16816(s[a], a1, kf[a][i].z, kf[a][i].w);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint4* src = sq + ((mt * KW + i) * 4) * 32 + lane;
          const uint4 h0 = src[0], h1 = src[32], l0 = src[64], l1 = src[96];
          uint32_t bh[4], bl[4];
          split_fast(__uint_as_float(kf[0][i].x), bh[0], bl[0]), split_fast(__uint_as_float(kf[0][i].y), bh[1], bl[1]);
          split_fast(__uint_as_float(kf[0][i].z), bh[2], bl[2]), split_fast(__uint_as_float(kf[0][i].w), bh[3], bl[3]);
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // short sums on the tensor cores, joined in fp32
          mma_1688(part, reinterpret_cast<const uint32_t*>(&l0), bh[0], bh[1]);
          mma_1688(part, reinterpret_cast<const uint32_t*>(&l1), bh[2], bh[3]);
          mma_1688(part, reinterpret_cast<const uint32_t*>(&h0), bl[0], bl[1]);
          mma_1688(part, reinterpret_cast<const uint32_t*>(&h1), bl[2], bl[3]);
          mma_1688(part, reinterpret_cast<const uint32_t*>(&h0), bh[0], bh[1]);
          mma_1688(part, reinterpret_cast<const uint32_t*>(&h1), bh[2], bh[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][e] += part[e];
        }
      }
      if (more) load_k(blk + KS, page_n);
      // online softmax in log2 units
      float mx_a = m_a, mx_b = m_b;
#pragma unroll
      for (int a = 0; a < KN; ++a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] *= p.scale_log2;
        if (key0 + KEYS > lim_0) {  // some row of the warp does not see the whole block
          const int key = key0 + 8 * a + 2 * t;
          if (key >= lim_a) s[a][0] = -INFINITY;
          if (key + 1 >= lim_a) s[a][1] = -INFINITY;
          if (key >= lim_b) s[a][2] = -INFINITY;
          if (key + 1 >= lim_b) s[a][3] = -INFINITY;
        }
        mx_a = fmax3(mx_a, s[a][0], s[a][1]);
        mx_b = fmax3(mx_b, s[a][2], s[a][3]);
      }
      mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
      mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
      mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
      mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
      if (__any_sync(0xffffffffu, mx_a > m_a || mx_b > m_b)) {
        const float fa = mx_a > m_a ? ex2(m_a - mx_a) : 1.0f, fb = mx_b > m_b ? ex2(m_b - mx_b) : 1.0f;
        l_a *= fa;
        l_b *= fb;
#pragma unroll
        for (int i = 0; i < NO; ++i) o[i][0] *= fa, o[i][1] *= fa, o[i][2] *= fb, o[i][3] *= fb;
        m_a = mx_a;
        m_b = mx_b;
      }
      const float ua = m_a == -INFINITY ? 0.0f : m_a, ub = m_b == -INFINITY ? 0.0f : m_b;
#pragma unroll
      for (int a = 0; a < KN; ++a) {
        s[a][0] = ex2(s[a][0] - ua);
        s[a][1] = ex2(s[a][1] - ua);
        s[a][2] = ex2(s[a][2] - ub);
        s[a][3] = ex2(s[a][3] - ub);
        l_a += s[a][0] + s[a][1];
        l_b += s[a][2] + s[a][3];
      }
      // O += P V
      if (HALF) {  // p in [0, 1] enters the product as fp16 (relative error 2^-12 at most; the sum l keeps fp32)
        const uint32_t pa[4] = {pack_half2(s[0][0], s[0][1]), pack_half2(s[0][2], s[0][3]),
                                pack_half2(s[KN - 1][0], s[KN - 1][1]), pack_half2(s[KN - 1][2], s[KN - 1][3])};
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const uint32_t* r0v = reinterpret_cast<const uint32_t*>(&vf[0][i]);
          const uint32_t* r1v = reinterpret_cast<const uint32_t*>(&vf[1][i]);
          const uint32_t* r2v = reinterpret_cast<const uint32_t*>(&vf[VN - 2][i]);
          const uint32_t* r3v = reinterpret_cast<const uint32_t*>(&vf[VN - 1][i]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
            mma_16816(o[8 * i + j], pa, __byte_perm(r0v[j >> 1], r1v[j >> 1], sel), __byte_perm(r2v[j >> 1], r3v[j >> 1], sel));
          }
        }
      } else {  // inner index t <-> key 2t, t + 4 <-> key 2t + 1
        uint32_t ph[4], pl[4];
        split_fast(s[0][0], ph[0], pl[0]), split_fast(s[0][2], ph[1], pl[1]);
        split_fast(s[0][1], ph[2], pl[2]), split_fast(s[0][3], ph[3], pl[3]);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const uint32_t* r0v = reinterpret_cast<const uint32_t*>(&vf[0][i]);
          const uint32_t* r1v = reinterpret_cast<const uint32_t*>(&vf[1][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t h0, h1, l0, l1;
            split_fast(__uint_as_float(r0v[j]), h0, l0), split_fast(__uint_as_float(r1v[j]), h1, l1);
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_1688(part, pl, h0, h1);
            mma_1688(part, ph, l0, l1);
            mma_1688(part, ph, h0, h1);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * i + j][e] += part[e];
          }
        }
      }
      if (more) load_v(blk + KS, page_n);
    }

    // ---- join the key shares
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    __syncthreads();  // the previous item's sums have been read
    if (t == 0) {
      sm.m[warp][g] = m_a, sm.m[warp][g + 8] = m_b;
      sm.l[warp][g] = l_a, sm.l[warp][g + 8] = l_b;
    }
    // column n = 2t + (e & 1) of output tile (i, j) is feature W i + (W / 8) n + j, W = 64 (fp16), 32 (fp32)
    constexpr int J = HALF ? 8 : 4;
#pragma unroll
    for (int i = 0; i < VW; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < J; j += 4) {
          const int col = i * J * 8 + J * (2 * t + e) + j;
          *reinterpret_cast<float4*>(&sm.o[warp][g][col]) =
              make_float4(o[J * i + j][e], o[J * i + j + 1][e], o[J * i + j + 2][e], o[J * i + j + 3][e]);
          *reinterpret_cast<float4*>(&sm.o[warp][g + 8][col]) =
              make_float4(o[J * i + j][2 + e], o[J * i + j + 1][2 + e], o[J * i + j + 2][2 + e], o[J * i + j + 3][2 + e]);
        }
    __syncthreads();
    const bool complete = tile0 == 0 && tiles == nt;
    const int slot = tile0 == 0 ? 1 : 0;  // 0: the item began before this CTA
    if (!complete && slot == 1 && tid == 0) {
      const int64_t last = base + (item + 1) * nt;  // one past the item's last tile
      const int64_t end = (last * ctas - 1) / total;
      p.part_item[blockIdx.x] = make_int4(n, head, rtile, static_cast<int>(end - blockIdx.x));
    }
    constexpr int CH = DB / 4;  // float4 columns of a row
    for (int idx = tid; idx < ROWS * CH; idx += kThreads) {
      const int row = idx / CH, c = (idx - row * CH) * 4;
      const int r = rtile * ROWS + row;
      if (r >= total_rows) continue;
      const int rm = row / kRows, rr = row - rm * kRows;
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < KS; ++k) m = fmaxf(m, sm.m[k * MT + rm][rr]);
      const float u = m == -INFINITY ? 0.0f : m;
      float l = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const float f = ex2(sm.m[k * MT + rm][rr] - u);
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[k * MT + rm][rr][c]);
        l = fmaf(sm.l[k * MT + rm][rr], f, l);
        acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
      }
      if (complete) {
        const int64_t orow = static_cast<int64_t>(sl.begin + r / p.G) * p.H_q + head * p.G + r % p.G;
        store_row<T>(p, orow, c, acc, m, l);
      } else {
        const int64_t prow = (static_cast<int64_t>(blockIdx.x) * 2 + slot) * ROWS + row;
        *reinterpret_cast<float4*>(p.part_o + prow * DB + c) = acc;
        if (c == 0) p.part_ml[prow] = make_float2(m, l);
      }
    }
    w += tiles;
  }
}

// Joins the pieces of the item that begins in CTA blockIdx.x and goes on in
// the next ones: a thread adds one float4 column of one row over them.
template <typename T, int DB, int MT>
__global__ void __launch_bounds__(kThreads) merge_kernel(const Params p) {
  constexpr int ROWS = kRows * MT, CH = DB / 4;
  pdl_launch_dependents();
  pdl_wait();
  const int4 it = p.part_item[blockIdx.x];  // sequence, head, row tile, further pieces
  if (it.w < 0) return;
  const SeqLens sl = seq_lens(p.view, it.x);
  const int idx = blockIdx.y * kThreads + threadIdx.x;
  const int row = idx / CH, c = (idx - row * CH) * 4, r = it.z * ROWS + row;
  if (r >= sl.count * p.G) return;
  // piece 0 is slot 1 of its CTA, the others are slot 0 of theirs
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 2 + 1) * ROWS + row, step = 2 * ROWS;
  const int64_t rest = first + ROWS;
  float2 ml = p.part_ml[first];
  float m = ml.x;
  for (int i = 0; i < it.w; ++i) m = fmaxf(m, p.part_ml[rest + i * step].x);
  const float u = m == -INFINITY ? 0.0f : m;
  float f = ex2(ml.x - u), l = ml.y * f;
  float4 acc = *reinterpret_cast<const float4*>(p.part_o + first * DB + c);
  acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll 4
  for (int i = 0; i < it.w; ++i) {
    const float2 a = p.part_ml[rest + i * step];
    const float4 x = *reinterpret_cast<const float4*>(p.part_o + (rest + i * step) * DB + c);
    const float w = ex2(a.x - u);
    l = fmaf(a.y, w, l);
    acc.x = fmaf(x.x, w, acc.x), acc.y = fmaf(x.y, w, acc.y);
    acc.z = fmaf(x.z, w, acc.z), acc.w = fmaf(x.w, w, acc.w);
  }
  store_row<T>(p, static_cast<int64_t>(sl.begin + r / p.G) * p.H_q + it.y * p.G + r % p.G, c, acc, m, l);
}

}  // namespace paged
}  // namespace sdpa_b200
