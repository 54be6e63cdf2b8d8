// Attention of new tokens over the paged cache, for sequences with few of
// them (single tokens, drafted ones) in fp16, and for all in fp32.
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j,   stats_i = max + ln(sum + 1e-6)
//
// Bound: the bytes of the K and V rows held, read once (each serves only the
// rows of its head group).  The G = H_q / H_kv query heads of a KV head and the
// sequence's new tokens are packed into rows r = token * G + g, 16 to a tile,
// so all of them share one reading.  The products go through warp-level
// matrix instructions (m16n8k16 fp16; m16n8k8 tf32 three times a product for
// fp32, the product of the two low parts, 2^-22 of it, left out; its tiles have 8
// rows up to 16 packed rows a sequence: see Shape): 16 rows are a tenth of a tcgen05
// tile, and its operands would have to pass through shared memory and TMEM, while
// these take them from registers.
//
// Every warp streams alone: TMA boxes of one block of keys (16 fp16, 8 fp32;
// always inside one page) go to the warp's own ring of kStages blocks in shared
// memory, 128-byte swizzled, so the matrix operands come out of it without
// bank conflicts (ldmatrix; for fp32 values 16-byte loads, four output columns
// a word), and no barrier of the CTA stands in the loop.  16 x 32768 keys x 4 heads x
// 128 fp16 take 183 us (5.9 TB/s).  Operands copied lane by lane took 450
// instructions a block of 16 keys instead of about 170, and 196 us (plain loads,
// two blocks' worth of registers) or 243 us (cp.async).
//
// Work: every (sequence, KV head, row tile) item has ceil(held / 32) tiles of
// 32 keys; the tiles of all items, in order, are cut into equal ranges, one a
// warp (with more than 16 packed rows a sequence, one a group of 2 or 4 warps
// with a row tile each), so long and short sequences load the device evenly.
// An item that lies in one range is finished there; one that is cut leaves
// partial sums, at most two a range, that merge_kernel joins (32 sequences of 64 to
// 8192 keys x 8 heads x 128: 74 us, about 4 of them the merge).
#pragma once
#include "common.cuh"
#include "fwd_tc.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace sdpa_b200 {
namespace paged {

constexpr int kTile = 32;       // keys of one unit of work
constexpr int kLeast = 2;       // tiles of a range
constexpr int kLong = 16;       // pieces behind the first from which an item is merged in kParts parts
constexpr int kParts = 4;
constexpr int kRows = 16;       // packed query rows of one matrix tile
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMergeThreads = 256;

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
  // workspace of the kernel for few rows: items cut between ranges
  float* part_o;          // [ranges, 2, part_rows, part_cols] unnormalised sums
  float2* part_ml;        // [ranges, 2, part_rows] (max, sum), log2 units
  int4* part_item;        // [ranges] of the item cut at the range's end: (its sequence's first token, its first
                          // packed row, its rows | part << 16, KV head << 16 | ranges behind its first that hold the
                          // rest); 0 rows: none.  The range that an item begins in has part 0; of one with many
                          // pieces the next ranges, inside it, have parts 1 to 3: four blocks merge its rows
  int part_ranges, part_rows, part_cols;
  // workspace of the chunk kernel: pieces of cut items
  float* tc_o;            // [slots, 256, DV]
  float2* tc_ml;          // [slots, 256]
  int4* tc_item;          // [slots] (the pair's first token, its tokens, KV head, pieces << 16 | this one's index)
  int* tc_slots;          // slots in use
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
// x = hi + lo, both tf32 values: hi is x rounded to 11 bits, by half a step added
// to its bits (a carry moves on into the exponent), lo the rest (exact) cut to
// 11.  Finite for |x| < 2^128 (1 - 2^-12).  A NaN stays one in lo, which every
// product takes part of, whatever its bits become in hi; an infinity gives NaN.
// (The conversion instruction runs at a fraction of the rate; splitting by the
// product with 2^13 + 1 takes one instruction more and overflows from 2^115 on.)
__device__ __forceinline__ void split_fast(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi))) & 0xffffe000u;
}
__device__ __forceinline__ void split_fast(const uint4& x, uint4& hi, uint4& lo) {
  split_fast(__uint_as_float(x.x), hi.x, lo.x);
  split_fast(__uint_as_float(x.y), hi.y, lo.y);
  split_fast(__uint_as_float(x.z), hi.z, lo.z);
  split_fast(__uint_as_float(x.w), hi.w, lo.w);
}

// Four 8 x 8 matrices of 16-bit elements (or 8 x 4 of 32-bit ones); lane i
// gives the row address of matrix i / 8, row i % 8.
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ int row_tiles(const Params& p, const SeqLens& s, int rows) {
  return static_cast<int>((static_cast<int64_t>(s.count) * p.G + rows - 1) / rows);
}
__device__ __forceinline__ int key_tiles(const SeqLens& s) { return s.held > 0 ? (s.held + kTile - 1) / kTile : 1; }

// Shapes of one instantiation.  DB: feature bucket; MT: row tiles (warps) of a
// group, which shares one ring.
//
// fp32 with one row tile is thin: 8 rows.  Q's low parts take rows 8-15 of the
// first product, so q_hi k + q_lo k is one instruction and Q K^T takes two
// a step, not three; the second product is O^T = V^T P^T, 16 features x 8 rows,
// whose P^T operand is the scores' own layout.  Half the sums' registers and no
// part of Q in shared memory let three CTAs of D = 128 on an SM, not two (32 x 8192 keys x
// 8 heads x 128, 4 rows: 336 us, 6.4 TB/s; about 40 us more with two, 160 with 16 rows).
template <typename T, int DB, int MT>
struct Shape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr bool kThin = !kHalf && MT == 1;
  static constexpr int kKeys = kHalf ? 16 : 8;              // keys of a block
  static constexpr int kBoxes = DB * static_cast<int>(sizeof(T)) / 128;  // 128-byte column boxes of K, and of V
  static constexpr int kBoxBytes = kKeys * 128;
  static constexpr int kStageBytes = 2 * kBoxes * kBoxBytes;  // 8 KB at DB = 128
  static constexpr int kCtas = DB == 64 || kThin ? 3 : 2;  // resident CTAs an SM
  static constexpr int kStages = (DB == 64 ? (kHalf ? 4 : 3) : (kHalf ? 3 : 2)) * MT;
  static constexpr int kGroups = kWarps / MT;               // ranges of a CTA
  static constexpr int kQBytes = kHalf || kThin ? 0 : DB / 8 * 512;  // a warp's low parts of Q (fp32)
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kSmemBytes = kGroups * kRingBytes + kWarps * kQBytes + 1024;  // + alignment slack
  static constexpr int kTileRows = kThin ? 8 : kRows;
  static constexpr int kRowsAll = kTileRows * MT;
};

// One output row's four columns from its sums (and, where asked, its stats):
// stats = max + ln(l + 1e-6); a row that saw no key is zero.
__device__ __forceinline__ float row_stats(float m, float l) {
  return (m == -INFINITY ? kNegInit : m * kLn2) + logf(l + kEps);
}
__device__ __forceinline__ float row_scale(float l) { return l <= kEps ? 0.0f : 1.0f / l; }  // (NaN stays)
template <typename T>
__device__ __forceinline__ void store4(T* dst, float x, float y, float z, float w) {
  if (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(x, y), pack_half2(z, w));
  else
    *reinterpret_cast<float4*>(dst) = make_float4(x, y, z, w);
}
template <typename T>
__device__ __forceinline__ void store_row(const Params& p, int64_t row, int c, const float4& acc, float m, float l) {
  const float inv = row_scale(l);
  if (c == 0) p.stats[row] = row_stats(m, l);
  if (c < p.D_v) store4<T>(static_cast<T*>(p.out) + row * p.D_v + c, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// (m, l, acc) += a piece's (max, sum) and sums.
__device__ __forceinline__ void join(float& m, float& l, float4& acc, const float2& ml, const float4& x) {
  const float up = fmaxf(m, ml.x), u = up == -INFINITY ? 0.0f : up;
  const float f = ex2(m - u), w = ex2(ml.x - u);
  m = up;
  l = fmaf(ml.y, w, l * f);
  acc.x = fmaf(x.x, w, acc.x * f), acc.y = fmaf(x.y, w, acc.y * f);
  acc.z = fmaf(x.z, w, acc.z * f), acc.w = fmaf(x.w, w, acc.w * f);
}

template <typename T, int DB, int MT>
__global__ void __launch_bounds__(kThreads, Shape<T, DB, MT>::kCtas)
    attend_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<T, DB, MT>;
  constexpr bool HALF = S::kHalf, THIN = S::kThin;
  constexpr int KEYS = S::kKeys, ST = S::kStages, BX = S::kBoxes;
  constexpr int KN = KEYS / 8;                 // score column tiles of a block
  constexpr int KS = HALF ? DB / 16 : DB / 8;  // inner steps of Q K^T
  constexpr int NO = THIN ? DB / 16 : DB / 8;  // output tiles
  constexpr int ROWS = S::kRowsAll;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = tc::align1024(smem_raw);
  __shared__ uint64_t s_full[S::kGroups * ST], s_empty[S::kGroups * ST];
  __shared__ int64_t s_warp[kWarps];
  __shared__ int64_t s_before[kThreads];  // tiles before thread i's sequences
  __shared__ int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mt = warp % MT, group = warp / MT;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* const ring = smem + group * S::kRingBytes;
  uint64_t* const full = s_full + group * ST;
  uint64_t* const empty = s_empty + group * ST;  // (used by groups of several warps)
  uint4* const q_lo = reinterpret_cast<uint4*>(smem + S::kGroups * S::kRingBytes + warp * S::kQBytes) + lane;  // fp32
  if (tid == 0) {
    for (int i = 0; i < S::kGroups * ST; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], MT);
    }
    s_abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_launch_dependents();
  pdl_wait();
  WaitCtl ctl;
  ctl.abort_flag = &s_abort;

  // ---- this group's range of tiles
  const int per = (p.view.seqs + kThreads - 1) / kThreads;
  int64_t mine = 0;
  bool descends = false;
  for (int n = tid * per; n < min(p.view.seqs, (tid + 1) * per); ++n) {
    const SeqLens s = seq_lens(p.view, n);
    descends |= !s.ascends;
    mine += static_cast<int64_t>(row_tiles(p, s, ROWS)) * key_tiles(s);
  }
  mine *= p.H_kv;
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) s_warp[warp] = incl;
  const bool refused = __syncthreads_or(descends) && seqs_overlap(p.view);
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  if (refused) total = 0;  // (see paged.cuh)
  s_before[tid] = before + incl - mine;
  __syncthreads();
  const int64_t range = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(gridDim.x) * group;
  // (fp16) fewer ranges where they would be short: one a warp scheduler, then kLeast tiles each
  const int64_t most = min(static_cast<int64_t>(gridDim.x) * S::kGroups, total);
  const int64_t ranges = HALF ? min(most, max(static_cast<int64_t>(4 * p.sms), total / kLeast)) : most;
  if (range >= ranges) {
    if (mt == 0 && lane == 0) p.part_item[range] = make_int4(0, 0, 0, 0);
    return;
  }
  const int64_t w0 = total * range / ranges, w1 = total * (range + 1) / ranges;
  // the last thread whose sequences begin at or before w0 (a chunk without work begins where the next does)
  int c = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) c += __popc(__ballot_sync(0xffffffffu, s_before[i * 32 + lane] <= w0));
  int n = (c - 1) * per;
  int64_t base = s_before[c - 1];
  int4 record = make_int4(0, 0, 0, 0);

  const int page_shift = p.view.page_shift, page_mask = (1 << page_shift) - 1;
  // this lane's row and 16-byte chunk in the ldmatrix loads of K and V (chunk ^ row % 8: the swizzle)
  const int sw = lane & 7, mi = lane >> 3;
  const uint32_t k_off = HALF ? ((mi >> 1) * 8 + sw) * 128 : sw * 128;
  const int k_chunk = HALF ? (mi & 1) : mi;
  const uint32_t v_off = HALF ? ((mi & 1) * 8 + sw) * 128 : 0;
  const int v_chunk = mi >> 1;
  int done = 0;  // blocks this group has taken through its ring
  bool ok = true;

  for (int64_t w = w0; w < w1 && ok;) {
    const SeqLens sl = seq_lens(p.view, n);
    const int rt = row_tiles(p, sl, ROWS), nt = key_tiles(sl);
    const int64_t work = static_cast<int64_t>(rt) * p.H_kv * nt;
    if (w >= base + work) {
      base += work;
      ++n;
      continue;
    }
    ctl.deadline_ns = globaltimer_ns() + p.timeout_ns;  // (of each item)
    const int64_t local = w - base;
    const int64_t item = local / nt;
    const int tile0 = static_cast<int>(local - item * nt);
    const int head = static_cast<int>(item / rt), rtile = static_cast<int>(item - static_cast<int64_t>(head) * rt);
    const int tiles = static_cast<int>(min(static_cast<int64_t>(nt - tile0), w1 - w));

    // ---- the blocks of keys, and their copies
    const int blk0 = tile0 * (kTile / KEYS);
    const int blocks = (min((tile0 + tiles) * kTile, sl.held) + KEYS - 1) / KEYS - blk0;
    // pages of 32 blocks, one a lane, read a batch ahead
    auto pages_from = [&](int i) {
      return i + lane < blocks ? page_of(p.view, n, ((blk0 + i + lane) * KEYS) >> page_shift) : -1;
    };
    int pages = -1, pages_next = -1;
    if (mt == 0) pages = pages_from(0), pages_next = pages_from(32);
    // Block i to its stage (whole warp; the group's first).  Features behind D
    // and pages outside the pool (-1) read as zeros.
    auto copy_block = [&](int i) {
      if (i > 0 && (i & 31) == 0) {
        pages = pages_next;
        pages_next = pages_from(i + 32);
      }
      const int page = __shfl_sync(0xffffffffu, pages, i & 31);
      if (lane == 0) {
        const int stage = (done + i) % ST;
        const int row = ((blk0 + i) * KEYS) & page_mask;
        uint8_t* const dst = ring + stage * S::kStageBytes;
        mbar_expect_tx(&full[stage], S::kStageBytes);
#pragma unroll
        for (int x = 0; x < BX; ++x)
          tma_load_4d(dst + x * S::kBoxBytes, &tm_k, x * (128 / static_cast<int>(sizeof(T))), head, row, page, &full[stage]);
#pragma unroll
        for (int x = 0; x < BX; ++x)
          tma_load_4d(dst + (BX + x) * S::kBoxBytes, &tm_v, x * (128 / static_cast<int>(sizeof(T))), head, row, page,
                      &full[stage]);
      }
    };
    int copied = 0;
    if (mt == 0)
      for (; copied < min(ST, blocks); ++copied) {
        // a group of several warps: all of them have left the stage's last block
        if (MT > 1 && !tc::warp_wait(&empty[(done + copied) % ST], (((done + copied) / ST) & 1) ^ 1, ctl)) {
          ok = false;
          break;
        }
        copy_block(copied);
      }

    // ---- rows of this warp
    const int total_rows = sl.count * p.G;
    const int r0 = (rtile * MT + mt) * S::kTileRows;
    const int ra = r0 + g, rb = r0 + g + 8;
    const bool va = ra < total_rows, vb = !THIN && rb < total_rows;
    const int shift = sl.held - sl.count;  // position of the first new token
    // keys a row sees: [0, lim)
    const int lim_a = p.causal ? min(sl.held, shift + ra / p.G + 1) : sl.held;
    const int lim_b = p.causal ? min(sl.held, shift + rb / p.G + 1) : sl.held;
    const int lim_0 = p.causal ? min(sl.held, shift + r0 / p.G + 1) : sl.held;  // the least of the warp's
    const T* qa = static_cast<const T*>(p.q) + (sl.begin + ra / p.G) * p.q_stride + (head * p.G + ra % p.G) * p.D;
    const T* qb = static_cast<const T*>(p.q) + (sl.begin + rb / p.G) * p.q_stride + (head * p.G + rb % p.G) * p.D;
    // A operands: (row g, k t) (row g+8, k t) (row g, k t') (row g+8, k t'); k t is a pair of halves or one float
    uint32_t qf[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const int d0 = HALF ? 16 * i + 2 * t : 8 * i + t, d1 = d0 + (HALF ? 8 : 4);
      qf[i][0] = va && d0 < p.D ? __ldg(reinterpret_cast<const uint32_t*>(qa + d0)) : 0u;
      qf[i][1] = vb && d0 < p.D ? __ldg(reinterpret_cast<const uint32_t*>(qb + d0)) : 0u;
      qf[i][2] = va && d1 < p.D ? __ldg(reinterpret_cast<const uint32_t*>(qa + d1)) : 0u;
      qf[i][3] = vb && d1 < p.D ? __ldg(reinterpret_cast<const uint32_t*>(qb + d1)) : 0u;
    }
    if (!HALF) {
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_fast(__uint_as_float(qf[i][e]), qf[i][e], lo[e]);
        if (THIN)
          qf[i][1] = lo[0], qf[i][3] = lo[2];
        else
          q_lo[i * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }

    float o[NO][4];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;

    for (int i = 0; ok && i < blocks; ++i) {
      const int key0 = (blk0 + i) * KEYS;
      const int stage = (done + i) % ST;
      uint8_t* const at = ring + stage * S::kStageBytes;
      const uint32_t k_at = smem_u32(at), v_at = k_at + BX * S::kBoxBytes;
      if (!tc::warp_wait(&full[stage], ((done + i) / ST) & 1, ctl)) {
        ok = false;
        break;
      }
      if (key0 + KEYS > sl.held) {
        // V rows behind the sequence count as zeros: whatever the pool holds there stays out of the sums
        for (int x = lane; x < BX * KEYS * 8; x += 32)
          if (key0 + (x >> 3) % KEYS >= sl.held)
            *reinterpret_cast<uint4*>(at + BX * S::kBoxBytes + x * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // before the stage's next copy
        __syncwarp();
      }
      // S = Q K^T
      float s[KN][4];
#pragma unroll
      for (int a = 0; a < KN; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] = 0.0f;
      if (HALF) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t b[4];  // keys 0-7 and 8-15, two operands each
          ldmatrix4(k_at + (k >> 2) * S::kBoxBytes + k_off + (((2 * (k & 3) + k_chunk) ^ sw) << 4), b);
          mma_16816(s[0], qf[k], b[0], b[1]);
          mma_16816(s[KN - 1], qf[k], b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; k += 4) {
          uint32_t b[2][4], bl[2][4];  // twice two inner steps, two operands each
          uint4 l[4];
          float part[2][4];  // short sums on the tensor cores, joined in fp32
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k2 = k + 2 * h;
            ldmatrix4(k_at + (k2 >> 2) * S::kBoxBytes + k_off + (((2 * (k2 & 3) + k_chunk) ^ sw) << 4), b[h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) split_fast(__uint_as_float(b[h][e]), b[h][e], bl[h][e]), part[h][e] = 0.0f;
            if (!THIN) l[2 * h] = q_lo[k2 * 32], l[2 * h + 1] = q_lo[(k2 + 1) * 32];
          }
          // two sums in turn: a product waits 21 cycles for the last one of its sum, 8 for another's
          if (!THIN) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mma_1688(part[h], reinterpret_cast<const uint32_t*>(&l[2 * h + x]), b[h][2 * x], b[h][2 * x + 1]);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) mma_1688(part[h], qf[k + 2 * h + x], bl[h][2 * x], bl[h][2 * x + 1]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) mma_1688(part[h], qf[k + 2 * h + x], b[h][2 * x], b[h][2 * x + 1]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][THIN ? e & 1 : e] += part[h][e];
        }
      }
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
          if (!THIN && key >= lim_b) s[a][2] = -INFINITY;
          if (!THIN && key + 1 >= lim_b) s[a][3] = -INFINITY;
        }
        mx_a = fmax3(mx_a, s[a][0], s[a][1]);
        if (!THIN) mx_b = fmax3(mx_b, s[a][2], s[a][3]);
      }
      mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
      if (!THIN) mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
      mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
      if (!THIN) mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
      if (__any_sync(0xffffffffu, mx_a > m_a || mx_b > m_b)) {
        float fa = mx_a > m_a ? ex2(m_a - mx_a) : 1.0f, fb = mx_b > m_b ? ex2(m_b - mx_b) : 1.0f;
        l_a *= fa;
        l_b *= fb;
        if (THIN) {  // the output's rows are 2t and 2t + 1
          fb = __shfl_sync(0xffffffffu, fa, 8 * t + 4);
          fa = __shfl_sync(0xffffffffu, fa, 8 * t);
        }
#pragma unroll
        for (int x = 0; x < NO; ++x)
          o[x][0] *= fa, o[x][1] *= THIN ? fb : fa, o[x][2] *= THIN ? fa : fb, o[x][3] *= fb;
        m_a = mx_a;
        m_b = mx_b;
      }
      const float ua = m_a == -INFINITY ? 0.0f : m_a, ub = m_b == -INFINITY ? 0.0f : m_b;
#pragma unroll
      for (int a = 0; a < KN; ++a) {
        s[a][0] = ex2(s[a][0] - ua);
        s[a][1] = ex2(s[a][1] - ua);
        l_a += s[a][0] + s[a][1];
        if (THIN) continue;  // (no rows g + 8)
        s[a][2] = ex2(s[a][2] - ub);
        s[a][3] = ex2(s[a][3] - ub);
        l_b += s[a][2] + s[a][3];
      }
      // O += P V
      if (HALF) {  // p in [0, 1] enters the product as fp16 (relative error 2^-11 at most; the sum l keeps fp32)
        const uint32_t pa[4] = {pack_half2(s[0][0], s[0][1]), pack_half2(s[0][2], s[0][3]),
                                pack_half2(s[KN - 1][0], s[KN - 1][1]), pack_half2(s[KN - 1][2], s[KN - 1][3])};
#pragma unroll
        for (int x = 0; x < NO; x += 2) {
          uint32_t b[4];  // two column tiles, keys 0-7 and 8-15 each
          ldmatrix4_trans(v_at + (x >> 3) * S::kBoxBytes + v_off + ((((x & 7) + v_chunk) ^ sw) << 4), b);
          mma_16816(o[x], pa, b[0], b[1]);
          mma_16816(o[x + 1], pa, b[2], b[3]);
        }
      } else {  // inner index t <-> key 2t, t + 4 <-> key 2t + 1; word g of a box row: column g of four tiles
        uint32_t ph[4], pl[4];
        split_fast(s[0][0], ph[0], pl[0]), split_fast(s[0][1], ph[2], pl[2]);
        if (!THIN) split_fast(s[0][2], ph[1], pl[1]), split_fast(s[0][3], ph[3], pl[3]);
#pragma unroll
        for (int x = 0; x < BX; ++x) {
          const uint8_t* box = at + (BX + x) * S::kBoxBytes;
          uint4 h0, l0, h1, l1;
          split_fast(*reinterpret_cast<const uint4*>(box + (2 * t) * 128 + ((g ^ (2 * t)) << 4)), h0, l0);
          split_fast(*reinterpret_cast<const uint4*>(box + (2 * t + 1) * 128 + ((g ^ (2 * t + 1)) << 4)), h1, l1);
          const uint32_t *xh0 = reinterpret_cast<const uint32_t*>(&h0), *xh1 = reinterpret_cast<const uint32_t*>(&h1);
          const uint32_t *xl0 = reinterpret_cast<const uint32_t*>(&l0), *xl1 = reinterpret_cast<const uint32_t*>(&l1);
          if (THIN) {  // tile 2x + j: features 32x + 4g + 2j (rows g) and + 1 (rows g + 8)
            float part[2][4] = {};
            const uint32_t a[2][4] = {{xh0[0], xh0[1], xh1[0], xh1[1]}, {xh0[2], xh0[3], xh1[2], xh1[3]}};
            const uint32_t al[2][4] = {{xl0[0], xl0[1], xl1[0], xl1[1]}, {xl0[2], xl0[3], xl1[2], xl1[3]}};
#pragma unroll
            for (int j = 0; j < 2; ++j) mma_1688(part[j], a[j], pl[0], pl[2]);
#pragma unroll
            for (int j = 0; j < 2; ++j) mma_1688(part[j], al[j], ph[0], ph[2]);
#pragma unroll
            for (int j = 0; j < 2; ++j) mma_1688(part[j], a[j], ph[0], ph[2]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[2 * x + j][e] += part[j][e];
            continue;
          }
          float part[4][4] = {};  // (four sums in turn, as above)
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_1688(part[j], pl, xh0[j], xh1[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_1688(part[j], ph, xl0[j], xl1[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_1688(part[j], ph, xh0[j], xh1[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * x + j][e] += part[j][e];
        }
      }
      __syncwarp();  // every lane has left the stage
      if (MT > 1 && lane == 0) mbar_arrive(&empty[stage]);
      if (mt == 0 && copied < blocks) {
        if (MT > 1 && !tc::warp_wait(&empty[stage], ((done + i) / ST) & 1, ctl)) {
          ok = false;
          break;
        }
        copy_block(copied++);
      }
    }
    if (!ok) {  // let copies in flight land before the CTA exits
      if (mt == 0 && lane == 0) {
        WaitCtl drain = ctl;
        drain.deadline_ns = globaltimer_ns() + p.timeout_ns;
        int dummy = 0;
        drain.abort_flag = &dummy;
        for (int i = max(0, copied - ST); i < copied; ++i) mbar_wait(&full[(done + i) % ST], ((done + i) / ST) & 1, drain);
      }
      break;
    }
    done += blocks;

    // ---- the item's sums, or this range's part of them
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
    const bool complete = tile0 == 0 && tiles == nt;
    const int slot = tile0 == 0 ? 1 : 0;  // 0: the item began before this range
    if (!complete && w + tiles == w1) {  // cut at the range's end
      const int64_t first_tile = base + item * nt;
      const int64_t first = slot == 1 ? range : ((first_tile + 1) * ranges - 1) / total;  // the range it began in
      const int more = static_cast<int>(((first_tile + nt) * ranges - 1) / total - first);
      const int part = static_cast<int>(range - first);
      if (part == 0 || (more >= kLong && part < kParts))
        record = make_int4(sl.begin, rtile * ROWS, min(ROWS, total_rows - rtile * ROWS) | part << 16, head << 16 | more);
    }
    const float inv_a = complete ? row_scale(l_a) : 1.0f, inv_b = complete ? row_scale(l_b) : 1.0f;
    const int64_t oa = static_cast<int64_t>(sl.begin + ra / p.G) * p.H_q + head * p.G + ra % p.G;
    const int64_t ob = static_cast<int64_t>(sl.begin + rb / p.G) * p.H_q + head * p.G + rb % p.G;
    const int64_t pa = (range * 2 + slot) * ROWS + mt * S::kTileRows + g, pb = pa + 8;
    if (t == 0) {
      if (complete) {
        if (va) p.stats[oa] = row_stats(m_a, l_a);
        if (vb) p.stats[ob] = row_stats(m_b, l_b);
      } else {
        if (va) p.part_ml[pa] = make_float2(m_a, l_a);
        if (vb) p.part_ml[pb] = make_float2(m_b, l_b);
      }
    }
    // Column n = 2t + e of output tile x: feature 8x + n (fp16), 32 (x / 4) + 4n + x % 4 (fp32).
    if (HALF) {
#pragma unroll
      for (int x = 0; x < NO; ++x) {
        const int col = 8 * x + 2 * t;
        if (complete) {
          if (col >= p.D_v) continue;
          if (va) *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + oa * p.D_v + col) = pack_half2(o[x][0] * inv_a, o[x][1] * inv_a);
          if (vb) *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + ob * p.D_v + col) = pack_half2(o[x][2] * inv_b, o[x][3] * inv_b);
        } else {
          if (va) *reinterpret_cast<float2*>(p.part_o + pa * DB + col) = make_float2(o[x][0], o[x][1]);
          if (vb) *reinterpret_cast<float2*>(p.part_o + pb * DB + col) = make_float2(o[x][2], o[x][3]);
        }
      }
    } else if (THIN) {  // rows 2t and 2t + 1; features as the product left them
      const float inv_0 = __shfl_sync(0xffffffffu, inv_a, 8 * t), inv_1 = __shfl_sync(0xffffffffu, inv_a, 8 * t + 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = r0 + 2 * t + e;
        if (row >= total_rows) continue;
        const float inv = e ? inv_1 : inv_0;
        float* const dst = complete ? static_cast<float*>(p.out) +
                                          (static_cast<int64_t>(sl.begin + row / p.G) * p.H_q + head * p.G + row % p.G) * p.D_v
                                    : p.part_o + (pa - g + 2 * t + e) * DB;
#pragma unroll
        for (int x = 0; x < BX; ++x) {
          const int col = 32 * x + 4 * g;
          if (!complete || col < p.D_v)
            store4<float>(dst + col, o[2 * x][e] * inv, o[2 * x][e + 2] * inv, o[2 * x + 1][e] * inv, o[2 * x + 1][e + 2] * inv);
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < NO; x += 4)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = 8 * x + 4 * (2 * t + e);
          if (complete && col >= p.D_v) continue;
          float* const da = complete ? static_cast<float*>(p.out) + oa * p.D_v + col : p.part_o + pa * DB + col;
          float* const db = complete ? static_cast<float*>(p.out) + ob * p.D_v + col : p.part_o + pb * DB + col;
          if (va) store4<float>(da, o[x][e] * inv_a, o[x + 1][e] * inv_a, o[x + 2][e] * inv_a, o[x + 3][e] * inv_a);
          if (vb) store4<float>(db, o[x][2 + e] * inv_b, o[x + 1][2 + e] * inv_b, o[x + 2][2 + e] * inv_b, o[x + 3][2 + e] * inv_b);
        }
    }
    w += tiles;
  }
  if (mt == 0 && lane == 0) p.part_item[range] = record;
}

// Joins the pieces of cut items (the item that begins in range i and goes on in
// the next ones), which go round the blocks in turn.  A thread adds float4
// columns of a row over the pieces, whose values it reads several at a time
// (latency bounds this kernel); for items of few rows over every (shares)-th
// piece, the shares joined in shared memory.

// Pieces at rows first, first + step, .. (count of them) of one float4 column.
// All offsets fit 32 bits (the workspace is some tens of MB).
template <int AHEAD>
__device__ __forceinline__ void join_pieces(const float* o, const float2* ml, int first, int step, int count, int cols,
                                            float& m, float& l, float4& acc) {
  for (; count > 0; count -= AHEAD, first += AHEAD * step) {
    float2 a[AHEAD];
    float4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < count) {
        a[i] = ml[first + i * step];
        x[i] = *reinterpret_cast<const float4*>(o + (first + i * step) * cols);
      }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < count) join(m, l, acc, a[i], x[i]);
  }
}

// Rows part, part + parts, .. of the item that began in range `range`.
template <typename T>
__device__ __forceinline__ void merge_range(const Params& p, int range, int part, int parts, const int4& it,
                                            float4* s_acc, float2* s_ml) {
  const int ROWS = p.part_rows, shift = p.part_cols == 64 ? 4 : 5;  // log2 of a row's float4 columns
  const int rows = (it.z - part + parts - 1) / parts, pieces = (it.w & 0xffff) + 1, head = it.w >> 16;
  // rows a round takes, and (where the item has fewer) shares of the pieces
  const int round = kMergeThreads >> shift, at_once = min(rows, round), shares = min(pieces, round / at_once);
  const int group = threadIdx.x >> shift, c = (threadIdx.x & ((1 << shift) - 1)) * 4;
  const int share = group / at_once, row_in = group - share * at_once;
  // piece 0 is slot 1 of its range, piece i slot 0 of range + i: rows (2 range + 1) ROWS, then 2 ROWS apart from + ROWS
  const int row0 = (range * 2 + 1) * ROWS;
  for (int i_row = row_in; i_row - row_in < rows; i_row += at_once) {
    const bool live = share < shares && i_row < rows;
    const int row = part + i_row * parts;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
      // pieces 1 + share, 1 + share + shares, .. and, of share 0, piece 0
      if (share == 0) join_pieces<1>(p.part_o + c, p.part_ml, row0 + row, 0, 1, p.part_cols, m, l, acc);
      join_pieces<8>(p.part_o + c, p.part_ml, row0 + row + ROWS + share * 2 * ROWS, shares * 2 * ROWS,
                     (pieces - 1 - share + shares - 1) / shares, p.part_cols, m, l, acc);
    }
    if (shares > 1) {  // (then one round takes all rows)
      __syncthreads();
      s_acc[threadIdx.x] = acc;
      s_ml[threadIdx.x] = make_float2(m, l);
      __syncthreads();
      if (share == 0)
        for (int i = 1; i < shares; ++i) {
          const int from = threadIdx.x + ((i * at_once) << shift);
          join(m, l, acc, s_ml[from], s_acc[from]);
        }
    }
    if (live && share == 0) {
      const int r = it.y + row, tok = r / p.G;
      store_row<T>(p, static_cast<int64_t>(it.x + tok) * p.H_q + head * p.G + r - tok * p.G, c, acc, m, l);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const Params p) {
  __shared__ float4 s_acc[kMergeThreads];
  __shared__ float2 s_ml[kMergeThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int stride = gridDim.x;
  constexpr int kAhead = 2;  // records a block reads at once
  for (int i0 = blockIdx.x; i0 < p.part_ranges; i0 += kAhead * stride) {
    int4 it[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) it[k] = i0 + k * stride < p.part_ranges ? p.part_item[i0 + k * stride] : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int part = it[k].z >> 16, parts = (it[k].w & 0xffff) >= kLong ? kParts : 1;
      it[k].z &= 0xffff;
      if (it[k].z > part) merge_range<T>(p, i0 + k * stride - part, part, parts, it[k], s_acc, s_ml);
    }
  }
}

}  // namespace paged
}  // namespace sdpa_b200
