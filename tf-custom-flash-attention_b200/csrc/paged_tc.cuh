// Attention of chunks of new tokens over the paged cache on the 5th-generation
// tensor cores, fp16 in, fp32 accumulate.
//
// Bound: the two products (2 seen keys (D + D_v) operations a row) and the
// exponentials (one a score, 16 a clock and SM).  One CTA = two 128-row tiles
// that share every K/V tile of 64 keys: a TMA warp for K and one for V, and an
// MMA warp and a softmax warpgroup a row tile.
//   - Rows are packed (token, head of the group): a tile is floor(128 / G)
//     tokens x G heads, so the G heads of a KV head share one reading of it;
//     Q comes as one box (64 columns, G heads, 1 KV head, tokens) a tile.
//   - A K/V tile is 64 / min(page, 64) boxes, one page each, one issued by each
//     lane of the TMA warp (a page's boxes need its table entry first; the
//     entries of the next tile are read a tile ahead).
//   - Two score buffers a row tile: S(i+1) is there when the softmax of tile i
//     ends, and PV(i), S(i+2) are issued while it works on i+1, so neither the
//     products nor the barriers between the warps (~300 cycles from an arrival
//     to the waiter) stand in its way.  TMEM, 512 columns: O 2 x 128, and for
//     each row tile two slots of 64 columns, where P (fp16, 32 columns) goes
//     over S.  With tiles of 128 keys there is room for one slot a row tile:
//     softmax (1900 cycles) and products (2100 with their waits) took turns,
//     4000 cycles a tile of 128 keys for D = 128 and for D = 64.
//   - Keys behind the sequence are masked, and their V rows set to zero in
//     shared memory before the product (0 * NaN is NaN).
//
// Work: an item is a pair of row tiles of one (sequence, KV head).  With at
// least as many items as SMs they run whole, but for the last items % SMs,
// which are cut into floor(SMs / rest) pieces each so that the last wave is
// full too.  With fewer, each is cut in proportion to its cost.  Pieces leave unnormalised sums that
// merge_kernel joins.  Every CTA works the cut out itself from the lengths on the device.
#pragma once
#include "fwd_tc.cuh"
#include "paged_mma.cuh"

namespace sdpa_b200 {
namespace paged_tc {

using paged::Params;
using tc::kBM;
using tc::warp_wait;

constexpr int kBN = 64;  // keys of a tile

constexpr int kThreads = 384;  // warps 0-7 softmax, 8 Q and K, 9 and 10 MMA, 11 V

// The MMA warps stay converged: every lane runs the loop and one elected lane
// issues, by a predicate on the instruction.  In a branch of one lane the
// compiler has to move every operand to the uniform registers that tcgen05
// takes: 870 cycles to issue eight MMAs, where their work is 256 (D = 64).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r));
  return r;
}
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(one)
      : "memory");
}

template <int DQK, int DV>
struct Cfg {
  static constexpr int kStages = 5;  // of the K ring and of the V ring
  static constexpr uint32_t kQBytes = kBM * DQK * 2;  // one row tile
  static constexpr uint32_t kKBytes = kBN * DQK * 2;
  static constexpr uint32_t kVBytes = kBN * DV * 2;
  static constexpr uint32_t kKOff = 2 * kQBytes;
  static constexpr uint32_t kVOff = kKOff + kStages * kKBytes;
  static constexpr uint32_t kBarOff = kVOff + kStages * kVBytes;
  static constexpr uint32_t kSmemBytes = kBarOff + 512 + 1024;  // + barriers + alignment slack
  static constexpr uint32_t kTmemCols = 512;
  static_assert(kSmemBytes <= 232448, "shared memory of a CTA");
};

struct Barriers {
  uint64_t q_full;
  uint64_t k_full[5], k_empty[5];
  uint64_t v_full[5], v_empty[5];
  uint64_t s_full[2][2];  // row tile, slot
  uint64_t p_full[2][2];
  uint64_t o_done[2];     // every PV of the row tile
  uint64_t o_final[2];    // its last
  uint64_t mma_done[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Barriers) <= 512, "barrier space");

constexpr int kPolyOf8 = 2;  // of 8 pairs of scores, those whose exponentials go to the FMA pipe
// 2^(r s + b) for two scores on the FMA pipe, for a part of the exponentials,
// to relieve the special function unit: x = n + f with n the nearest integer
// (by the addition of 1.5 * 2^23), |f| <= 1/2, 2^f by a polynomial of degree 4
// (least squares at Chebyshev nodes; off by 4e-6 at most, a sixtieth of the
// rounding of P to fp16), times 2^n.  x below -126 gives 2^-126,
// which fp16 rounds to zero.
__device__ __forceinline__ void exp2_pair(float& p0, float& p1, float r0, float r1, float s, float b) {
  float x0, x1, n0, n1, f0, f1;
  ffma2(x0, x1, r0, r1, s, s, b, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-126.0f));  // (a NaN score stays one)
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-126.0f));
  constexpr float kMagic = 12582912.0f;
  n0 = kMagic, n1 = kMagic;
  fadd2(n0, n1, x0, x1);
  float m0 = -kMagic, m1 = -kMagic;
  fadd2(m0, m1, n0, n1);                                   // n
  ffma2(f0, f1, m0, m1, -1.0f, -1.0f, x0, x1);             // f
  ffma2(p0, p1, f0, f1, 0.00957010128f, 0.00957010128f, 0.0559178591f, 0.0559178591f);
  ffma2(p0, p1, p0, p1, f0, f1, 0.240247443f, 0.240247443f);
  ffma2(p0, p1, p0, p1, f0, f1, 0.693121791f, 0.693121791f);
  ffma2(p0, p1, p0, p1, f0, f1, 0.999999285f, 0.999999285f);
  fmul2(p0, p1, p0, p1, __uint_as_float((__float_as_uint(n0) << 23) + 0x3f800000u),
        __uint_as_float((__float_as_uint(n1) << 23) + 0x3f800000u));  // 2^n, exactly
}

// Whether three barriers have all passed (one vote: 75 cycles; three waits one
// after the other, each for a phase long over, take 280).
__device__ __forceinline__ bool test3(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
      "and.pred p, p, q;\n\tand.pred p, p, r;\n\t"
      "vote.sync.all.pred p, p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(a)), "r"(pa), "r"(smem_u32(b)), "r"(pb), "r"(smem_u32(c)), "r"(pc)
      : "memory");
  return ok != 0;
}

// ---------------------------------------------------------------- the cut
struct Piece {
  int seq, head, pair;  // item
  int piece, pieces;    // its share of the item's keys
  int slot;             // workspace slot (pieces > 1)
};

__device__ __forceinline__ int pairs_of(const SeqLens& s, int tokens2) { return (s.count + tokens2 - 1) / tokens2; }
__device__ __forceinline__ int tiles_of(const SeqLens& s) { return max(1, (s.held + kBN - 1) / kBN); }

// Time of one of its items: a tile of 64 keys takes 1.10 us for a pair of row
// tiles, 0.70 us where the tokens fill the first alone (D = 128; 0.90 and 0.66 us
// for D = 64).
__device__ __forceinline__ float cost_of(const SeqLens& s, int tokens2) {
  return static_cast<float>(tiles_of(s)) * (s.count > tokens2 / 2 ? 9.0f : 6.0f);
}
constexpr float kStart = 54.0f;  // what a piece costs beside its tiles
// Pieces of an item: its cost in quanta, rounded (a piece costs from 2/3 to 3/2
// of a quantum), and no more than its tiles.
__device__ __forceinline__ int cuts_of(const SeqLens& s, int tokens2, float per_quantum) {
  return max(1, min(tiles_of(s), static_cast<int>(cost_of(s, tokens2) * per_quantum + 0.5f)));
}

__device__ __forceinline__ int warp_scan(int x) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, x, d);
    if ((threadIdx.x & 31) >= d) x += up;
  }
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}

// The piece that CTA `idx` computes; false if there is none.  Every warp works
// it out for itself (no barrier, and the same everywhere): lane i takes the
// i-th share of the sequences.  slots: workspace slots of the call.  (Items and
// pieces are counted in 32 bits and launched as CTAs; the host bounds both by the
// call's tokens and sequences, which holds while no two sequences share tokens:
// where they do there are no pieces and no slots, see paged.cuh.)
__device__ __forceinline__ bool find_piece(const Params& p, int idx, Piece& out, int& slots) {
  const int lane = threadIdx.x & 31;
  const int tokens2 = 2 * (kBM / p.G);
  const int per = (p.view.seqs + 31) / 32, n0 = lane * per, n1 = min(p.view.seqs, n0 + per);
  const SeqLens none = {0, 0, 0, true};
  const SeqLens s0 = n0 < n1 ? seq_lens(p.view, n0) : none;  // (the only one, up to 32 sequences)
  auto lens = [&](int n) { return n == n0 ? s0 : seq_lens(p.view, n); };
  int items = 0;
  bool descends = false;
  for (int n = n0; n < n1; ++n) {
    const SeqLens s = lens(n);
    items += pairs_of(s, tokens2);
    descends |= !s.ascends;
  }
  slots = 0;
  if (__any_sync(0xffffffffu, descends) && seqs_overlap(p.view)) return false;
  const int items_to = warp_scan(items);
  const int all_items = __shfl_sync(0xffffffffu, items_to, 31) * p.H_kv;
  const bool whole = all_items >= p.sms;  // the first `full` items run whole
  int target = idx, at = (items_to - items) * p.H_kv;  // first item (piece) of this lane's sequences
  int full = 0, cut = 1, piece = 0;
  float per_quantum = 0.0f;
  if (whole) {
    const int rest = all_items % p.sms;
    full = all_items - rest;
    const int cuts = rest ? p.sms / rest : 1;
    slots = cuts > 1 ? rest * cuts : 0;
    if (idx >= full) {
      cut = cuts;
      target = full + (idx - full) / cut;
      piece = (idx - full) % cut;
    }
  } else {
    float work = 0.0f;
    for (int n = n0; n < n1; ++n) work += static_cast<float>(pairs_of(lens(n), tokens2)) * cost_of(lens(n), tokens2);
    const float heads = static_cast<float>(p.H_kv), sms = static_cast<float>(p.sms);
    const float all = warp_sum(work) * heads;
    // The quantum, from 4/5 to 2 even shares of the SMs, whose pieces are
    // expected to end first: in one wave, the longest piece; in more, an even
    // share and half a piece.
    float best = INFINITY;
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      const float pq = sms / (all * (k == 0 ? 0.8f : k == 1 ? 1.0f : k == 2 ? 1.3f : 2.0f));
      float pieces = 0.0f, longest = 0.0f;
      for (int n = n0; n < n1; ++n) {
        const SeqLens s = lens(n);
        const float cuts = static_cast<float>(cuts_of(s, tokens2, pq));
        pieces += static_cast<float>(pairs_of(s, tokens2)) * cuts;
        if (s.count > 0) longest = fmaxf(longest, __fdividef(cost_of(s, tokens2), cuts));
      }
      pieces = warp_sum(pieces) * heads;
      float time = warp_max(longest) + kStart;
      if (pieces > sms) time = fmaxf(time, __fdividef(all + pieces * kStart, sms) + 0.5f * (__fdividef(all, pieces) + kStart));
      if (time < best) best = time, per_quantum = pq;
    }
    int mine = 0;
    float cost = 0.0f;
    for (int n = n0; n < n1; ++n) {
      const int cuts = cuts_of(lens(n), tokens2, per_quantum);
      mine += pairs_of(lens(n), tokens2) * cuts;
      cost = __fdividef(cost_of(lens(n), tokens2), static_cast<float>(cuts));
    }
    const int to = warp_scan(mine);
    slots = __shfl_sync(0xffffffffu, to, 31) * p.H_kv;
    at = to - mine;
    if (per == 1 && p.view.seqs > 1) {  // a sequence a lane: the longest pieces first, so that short ones fill the last gaps
      at = 0;
      for (int k = 0; k < p.view.seqs; ++k) {
        const float c = __shfl_sync(0xffffffffu, cost, k);
        const int m = __shfl_sync(0xffffffffu, mine, k);
        if (c > cost || (c == cost && k < lane)) at += m;
      }
    }
    at *= p.H_kv;
  }
  bool found = false;
  Piece f = {0, 0, 0, 0, 1, 0};
  for (int n = n0; n < n1; ++n) {
    const int pr = pairs_of(lens(n), tokens2);
    if (!whole) cut = cuts_of(lens(n), tokens2, per_quantum);
    const int count = pr * p.H_kv * (whole ? 1 : cut);
    if (target >= at && target < at + count) {
      int local = target - at;
      if (!whole) {
        piece = local % cut;
        local /= cut;
      }
      f.seq = n;
      f.head = local / pr;
      f.pair = pr - 1 - (local - f.head * pr);  // longest causal rows first
      f.piece = piece;
      f.pieces = cut;
      found = true;
    }
    at += count;
  }
  const unsigned who = __ballot_sync(0xffffffffu, found);
  if (!who) return false;
  const int src = __ffs(who) - 1;
  out.seq = __shfl_sync(0xffffffffu, f.seq, src);
  out.head = __shfl_sync(0xffffffffu, f.head, src);
  out.pair = __shfl_sync(0xffffffffu, f.pair, src);
  out.piece = __shfl_sync(0xffffffffu, f.piece, src);
  out.pieces = __shfl_sync(0xffffffffu, f.pieces, src);
  out.slot = idx - full;
  return true;
}

// Keys [0, lim) that token i (of the sequence's new ones) sees.
__device__ __forceinline__ int limit_of(const Params& p, const SeqLens& s, int i) {
  return p.causal ? max(0, min(s.held, s.held - s.count + i + 1)) : s.held;
}

// Key tiles of the item's pair of row tiles, and of this piece: [j0, j1).
struct Range {
  int tok0;      // first token of the pair (of the sequence's new ones)
  int n_item;    // key tiles the pair needs
  int j0, j1;
};
__device__ __forceinline__ Range range_of(const Params& p, const SeqLens& s, const Piece& w) {
  const int tokens2 = 2 * (kBM / p.G);
  Range r;
  r.tok0 = w.pair * tokens2;
  const int last = min(s.count, r.tok0 + tokens2) - 1;
  r.n_item = (limit_of(p, s, last) + kBN - 1) / kBN;
  r.j0 = static_cast<int>(static_cast<int64_t>(r.n_item) * w.piece / w.pieces);
  r.j1 = static_cast<int>(static_cast<int64_t>(r.n_item) * (w.piece + 1) / w.pieces);
  return r;
}

template <int DQK, int DV>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using C = Cfg<DQK, DV>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  Barriers* bars = reinterpret_cast<Barriers*>(smem + C::kBarOff);
  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 2);  // both MMA warps
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(&bars->s_full[t][s], 1);
        mbar_init(&bars->p_full[t][s], kBM);
      }
      mbar_init(&bars->o_done[t], 1);
      mbar_init(&bars->o_final[t], 1);
      mbar_init(&bars->mma_done[t], 1);
    }
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();  // (the barriers are set up)
  pdl_launch_dependents();
  pdl_wait();  // before any global access and before the wait deadline starts
  Piece w;
  int slots;
  const bool live = find_piece(p, static_cast<int>(blockIdx.x), w, slots);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.tc_slots = slots;
  if (!live) return;
  WaitCtl ctl;
  ctl.deadline_ns = globaltimer_ns() + p.timeout_ns;
  ctl.abort_flag = &bars->abort_flag;
  uint32_t tmem = 0;
  if (warp == 9) tmem_alloc(&bars->tmem_base, C::kTmemCols);
  if (warp != 8 && warp != 11) {  // (the TMA warps go ahead)
    tc_fence_before();
    asm volatile("bar.sync 1, 320;" ::: "memory");
    tc_fence_after();
    tmem = bars->tmem_base;
  }
  const SeqLens sl = seq_lens(p.view, w.seq);
  const Range rg = range_of(p, sl, w);
  const int tpt = kBM / p.G;  // tokens of a row tile
  // what merge_kernel goes by, of each slot
  if (threadIdx.x == 0 && w.slot >= 0 && w.slot < slots)
    p.tc_item[w.slot] = make_int4(sl.begin + rg.tok0, min(2 * tpt, sl.count - rg.tok0), w.head,
                                  w.pieces << 16 | w.piece);
  const int n_kv = rg.j1 - rg.j0;
  // key tiles per row tile within the piece; the second tile may have no tokens
  int n_t[2];
  {
    const int last_a = min(sl.count, rg.tok0 + tpt) - 1;
    n_t[0] = max(0, min(n_kv, (limit_of(p, sl, last_a) + kBN - 1) / kBN - rg.j0));
    n_t[1] = rg.tok0 + tpt < sl.count ? n_kv : 0;
  }

  if (warp == 8 || warp == 11) {
    // ------------------------------------- TMA: K (and Q) by warp 8, V by warp 11
    if (n_kv > 0) {
      const bool is_k = warp == 8;
      const int box = min(kBN, 1 << p.view.page_shift);
      const int subs = kBN / box;                    // boxes of a column block
      const int chunks = is_k ? DQK / 64 : DV / 64;  // column blocks
      const int sub = lane % subs, chunk = lane / subs;  // this lane's box (at most 4 x 2)
      const bool mine = chunk < chunks;
      const int page_mask = (1 << p.view.page_shift) - 1;
      const CUtensorMap* const map = is_k ? &tm_k : &tm_v;
      uint64_t* const full = is_k ? bars->k_full : bars->v_full;
      uint64_t* const empty = is_k ? bars->k_empty : bars->v_empty;
      const uint32_t stage_bytes = is_k ? C::kKBytes : C::kVBytes;
      uint8_t* const dst0 = smem + (is_k ? C::kKOff : C::kVOff) + chunk * kBN * 128 + sub * box * 128;
      if (lane == 0) {
        tma_prefetch_desc(map);
        if (is_k) {
          tma_prefetch_desc(&tm_q);
          // boxes of tpt tokens x G heads: tpt * G rows of each tile
          mbar_expect_tx(&bars->q_full, 2u * static_cast<uint32_t>(DQK / 64 * tpt * p.G * 128));
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < DQK / 64; ++c)
              tma_load_4d(smem + t * C::kQBytes + c * kBM * 128, &tm_q, c * 64, 0, w.head, sl.begin + rg.tok0 + t * tpt,
                          &bars->q_full);
        }
      }
      auto page_at = [&](int j) {
        const int key = (rg.j0 + j) * kBN + sub * box;
        return mine && j < n_kv && key < sl.held ? page_of(p.view, w.seq, key >> p.view.page_shift) : -1;
      };
      int page = page_at(0), issued = 0, s = 0;
      uint32_t phase = 1;
      for (int j = 0; j < n_kv; ++j) {
        const int next = page_at(j + 1);
        const int key0 = (rg.j0 + j) * kBN;
        const int boxes = min(subs, (sl.held - key0 + box - 1) / box);  // boxes that hold keys of the sequence
        if (!warp_wait(&empty[s], phase, ctl)) break;
        if (lane == 0) mbar_expect_tx(&full[s], static_cast<uint32_t>(chunks * boxes * box * 128));
        __syncwarp();
        if (mine && sub < boxes)  // a page id outside the pool (-1) reads as zeros
          tma_load_4d(dst0 + s * stage_bytes, map, chunk * 64, w.head, (key0 + sub * box) & page_mask, page, &full[s]);
        issued = j + 1;
        page = next;
        if (++s == ST) s = 0, phase ^= 1;
      }
      __syncwarp();
      if (*ctl.abort_flag && lane == 0) {  // let copies in flight land before the CTA exits
        WaitCtl drain = ctl;
        drain.deadline_ns = globaltimer_ns() + p.timeout_ns;
        int dummy = 0;
        drain.abort_flag = &dummy;
        if (is_k) mbar_wait(&bars->q_full, 0, drain);
        for (int j = max(0, issued - ST); j < issued; ++j) mbar_wait(&full[j % ST], (j / ST) & 1, drain);
      }
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------------------- MMA issuer of row tile t
    if (n_kv > 0) {
      constexpr uint32_t idesc_qk = make_idesc(kBM, kBN, false, false, false);
      constexpr uint32_t idesc_pv = make_idesc(kBM, DV, false, true, false);
      const int t = warp - 9, n_my = t ? n_t[1] : n_t[0];
      const uint32_t one = elect_one();
      // descriptors of stage 0; an offset of n bytes adds n / 16
      const uint64_t q_desc = make_sw128_desc(smem_u32(smem + t * C::kQBytes), 16, 1024);
      const uint64_t k_desc = make_sw128_desc(smem_u32(smem + C::kKOff), 16, 1024);
      const uint64_t v_desc = make_sw128_desc(smem_u32(smem + C::kVOff), kBN * 128, 1024);
      const uint32_t tO = tmem + t * 128, tS = tmem + 256 + t * 128;
      int ks = 0, vs = 0;  // stage of the next K and V tile, and their phases
      uint32_t kph = 0, vph = 0;
      auto issue_s = [&](int j) {  // S(j) = Q K_j^T, to slot j % 2; K_j is there
        if (j < n_my) {
#pragma unroll
          for (int kk = 0; kk < DQK / 16; ++kk) {
            const uint32_t in = (kk & 3) * 32;
            mma_ss(one, tS + (j & 1) * kBN, q_desc + ((kk >> 2) * (kBM * 128) + in) / 16,
                   k_desc + (ks * C::kKBytes + (kk >> 2) * (kBN * 128) + in) / 16, idesc_qk, kk > 0 ? 1u : 0u);
          }
          commit(one, &bars->s_full[t][j & 1]);
        }
        commit(one, &bars->k_empty[ks]);  // (an arrival alone where this row tile does not need the tile)
        if (++ks == ST) ks = 0, kph ^= 1;
      };
      bool ok = warp_wait(&bars->q_full, 0, ctl);
      for (int j = 0; ok && j < min(2, n_kv); ++j) {
        ok = warp_wait(&bars->k_full[ks], kph, ctl);
        tc_fence_after();
        if (ok) issue_s(j);
      }
      for (int j = 0; ok && j < n_kv; ++j) {
        // V_j, K_{j+2} (where there is one) and P(j) (where this row tile needs V_j)
        uint64_t* const vb = &bars->v_full[vs];
        uint64_t* const kb = j + 2 < n_kv ? &bars->k_full[ks] : vb;
        uint64_t* const pb = j < n_my ? &bars->p_full[t][j & 1] : vb;
        const uint32_t kp = j + 2 < n_kv ? kph : vph, pp = j < n_my ? (j >> 1) & 1 : vph;
        if (!test3(vb, vph, kb, kp, pb, pp) &&
            (!warp_wait(vb, vph, ctl) || !warp_wait(kb, kp, ctl) || !warp_wait(pb, pp, ctl))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (j < n_my) {
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)  // O += P(j) V_j
            mma_ts(one, tO, tS + (j & 1) * kBN + kk * 8, v_desc + (vs * C::kVBytes + kk * 16 * 128) / 16, idesc_pv,
                   (j > 0 || kk > 0) ? 1u : 0u);
          commit(one, &bars->o_done[t]);
          if (j == n_my - 1) commit(one, &bars->o_final[t]);
        }
        commit(one, &bars->v_empty[vs]);
        if (++vs == ST) vs = 0, vph ^= 1;
        if (j + 2 < n_kv) issue_s(j + 2);
      }
      commit(one, &bars->mma_done[t]);  // every MMA issued so far must finish before TMEM is released
      WaitCtl drain = ctl;
      drain.deadline_ns = globaltimer_ns() + p.timeout_ns;
      int dummy = 0;
      drain.abort_flag = &dummy;
      if (lane == 0) mbar_wait(&bars->mma_done[t], 0, drain);
    }
  } else {
    // ------------------------------------------------ softmax warpgroups
    const int t = warp >> 2;          // row tile of this warpgroup
    const int wq = warp & 3;          // TMEM lane quadrant
    const int r_in = wq * 32 + lane;  // TMEM lane = packed row of the tile
    const uint32_t lane_base = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tO = tmem + lane_base + t * 128;
    const int tok = rg.tok0 + t * tpt + r_in / p.G;  // of the sequence's new tokens
    const bool active = r_in < tpt * p.G && tok < sl.count;
    const bool warp_active = __any_sync(0xffffffffu, active);
    // rows without a token take no part: whatever they hold stays in their TMEM lane
    const int lim = active ? limit_of(p, sl, tok) : sl.held;
    const int lim_w = __shfl_sync(0xffffffffu, lim, 0);  // the least of the warp's
    const int n_my = n_t[t];
    const bool fold = p.scale_log2 > 0.0f;  // scale folded into one FFMA (max over raw scores)
    const float scl = fold ? p.scale_log2 : 1.0f;
    float m_run = -INFINITY;  // true running max (log2 units, scaled)
    float m_use = -INFINITY;  // reference max the exponentials are taken against
    float l = 0.0f;           // sum of exp2(x - m_use)
    bool ok = true;
    const uint32_t tS0 = tmem + lane_base + 256 + t * 128;
    auto step = [&](int j) -> bool {  // softmax of tile j
      uint32_t r[kBN];
      if (!warp_wait(&bars->s_full[t][j & 1], (j >> 1) & 1, ctl)) return false;
      tc_fence_after();
      SDPA_TMEM_LD32(tS0 + (j & 1) * kBN, (r + 0));
      SDPA_TMEM_LD32(tS0 + (j & 1) * kBN + 32, (r + 32));
      tmem_wait_ld();
      if ((rg.j0 + j + 1) * kBN > lim_w || !fold) {  // some row does not see the whole tile, or a scale <= 0
        const int left = max(0, min(kBN, lim - (rg.j0 + j) * kBN));
#pragma unroll
        for (int c = 0; c < kBN; ++c) {
          const float x = __uint_as_float(r[c]);
          r[c] = __float_as_uint(c >= left ? -INFINITY : fold ? x : x * p.scale_log2);
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four independent chains
#pragma unroll
      for (int c = 0; c < kBN; c += 8)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mx[q] = fmax3(mx[q], __uint_as_float(r[c + 2 * q]), __uint_as_float(r[c + 2 * q + 1]));
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scl;
      m_run = fmaxf(m_run, tmax);
      float alpha = 1.0f;
      bool rescale_o = false;
      if (tmax > m_use + tc::kRescaleThreshold) {
        alpha = ex2(m_use - m_run);  // 0 when m_use = -inf
        rescale_o = (j > 0) && (m_use != -INFINITY);
        m_use = m_run;
        l *= alpha;
      }
      const float nmu = (m_use == -INFINITY) ? 0.0f : -m_use;
      float rs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kBN; c += 2) {
        float p0, p1;
        if (c / 2 % 8 < kPolyOf8) {
          exp2_pair(p0, p1, __uint_as_float(r[c]), __uint_as_float(r[c + 1]), scl, nmu);
        } else {
          p0 = ex2(fmaf(__uint_as_float(r[c]), scl, nmu));
          p1 = ex2(fmaf(__uint_as_float(r[c + 1]), scl, nmu));
        }
        rs[(c >> 1) & 3] += p0 + p1;
        r[c / 2] = pack_half2(p0, p1);  // p <= 2^8 enters the product as fp16; the sum l keeps fp32
      }
      l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      SDPA_TMEM_ST32(tS0 + (j & 1) * kBN, r);
      if (__any_sync(0xffffffffu, rescale_o)) {
        // PV(j-1) must have finished (it may still run), PV(j) waits for this warp
        if (!warp_wait(&bars->o_done[t], (j - 1) & 1, ctl)) return false;
        tc_fence_after();
        const float a = rescale_o ? alpha : 1.0f;
#pragma unroll
        for (int c = 0; c < DV / 32; ++c) {
          uint32_t o[32];
          SDPA_TMEM_LD32(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
          SDPA_TMEM_ST32(tO + c * 32, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars->p_full[t][j & 1]);
      return true;
    };
    // V_j's rows behind the sequence are cleared before its product (thread r: row r; by both row tiles, whose
    // products are not ordered)
    auto clear_v = [&](int j) -> bool {
      const int s = j % ST;
      if (!warp_wait(&bars->v_full[s], (j / ST) & 1, ctl)) return false;
      if (r_in < kBN && (rg.j0 + j) * kBN + r_in >= sl.held) {
#pragma unroll
        for (int c = 0; c < DV / 64; ++c) {
          uint4* row = reinterpret_cast<uint4*>(smem + C::kVOff + s * C::kVBytes + c * kBN * 128 + r_in * 128);
#pragma unroll
          for (int e = 0; e < 8; ++e) row[e] = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      return true;
    };
    const int j_clear = n_my > 0 && (rg.j0 + n_my) * kBN > sl.held ? n_my - 1 : -1;  // the tile that holds the last key
    if (warp_active) {
      for (int j = 0; ok && j < n_my; ++j) {
        if (j == j_clear) ok = clear_v(j);
        if (ok) ok = step(j);
      }
    } else {  // no row of this warp has a token: it only keeps the barriers' counts
      for (int j = 0; ok && j < n_my; ++j) {
        if (j == j_clear) ok = clear_v(j);
        if (ok) ok = warp_wait(&bars->s_full[t][j & 1], (j >> 1) & 1, ctl);
        if (ok) mbar_arrive(&bars->p_full[t][j & 1]);
      }
    }
    // ----------------------------------------------------------- epilogue
    if (ok && n_my > 0) ok = warp_wait(&bars->o_final[t], 0, ctl);
    if (ok && warp_active) {
      tc_fence_after();
      const float f = m_run == -INFINITY ? 0.0f : ex2(m_use - m_run);
      const float l_true = l * f;  // relative to the true max
      const int64_t row = static_cast<int64_t>(sl.begin + tok) * p.H_q + w.head * p.G + r_in % p.G;
      const int64_t prow = static_cast<int64_t>(w.slot) * (2 * kBM) + t * kBM + r_in;
      const bool part = w.pieces > 1;
      const float mul = part ? f : (l_true <= kEps ? 0.0f : f / l_true);  // (NaN stays)
      if (active) {
        if (part)
          p.tc_ml[prow] = make_float2(m_run, l_true);
        else
          p.stats[row] = (m_run == -INFINITY ? kNegInit : m_run * kLn2) + logf(l_true + kEps);
      }
#pragma unroll
      for (int c = 0; c < DV / 32; ++c) {
        uint32_t o[32];
        if (n_my > 0) {
          SDPA_TMEM_LD32(tO + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        // a row that saw no key has no sum to scale (its O lane may hold anything)
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = mul == 0.0f ? 0.0f : __uint_as_float(o[e]) * mul;
        if (active) {
          if (part) {
            float4* dst = reinterpret_cast<float4*>(p.tc_o + prow * DV + c * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
          } else {
            __half* dst = static_cast<__half*>(p.out) + row * p.D_v + c * 32;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c * 32 + e * 8 < p.D_v)
                *reinterpret_cast<uint4*>(dst + e * 8) =
                    make_uint4(pack_half2(x[8 * e], x[8 * e + 1]), pack_half2(x[8 * e + 2], x[8 * e + 3]),
                               pack_half2(x[8 * e + 4], x[8 * e + 5]), pack_half2(x[8 * e + 6], x[8 * e + 7]));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the pieces of cut items: every slot's share of its item's rows, in
// quarters, go round the blocks in turn.
template <int DV>
__global__ void __launch_bounds__(paged::kMergeThreads) merge_kernel(const Params p) {
  constexpr int kRowsOfItem = 2 * kBM, CH = DV / 4;
  pdl_launch_dependents();
  pdl_wait();
  const int c = (threadIdx.x % CH) * 4;
  const int units = *p.tc_slots * 4, tpt = kBM / p.G;
  const float inv = 1.0f / static_cast<float>(p.G);
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int slot = u / 4;
    const int4 it = p.tc_item[slot];
    const int pieces = it.w >> 16, mine = it.w & 0xffff;
    if (pieces < 2) continue;
    const int parts = 4 * pieces, part = 4 * mine + u % 4;
    const int begin = kRowsOfItem * part / parts, end = kRowsOfItem * (part + 1) / parts;
    for (int row = begin + threadIdx.x / CH; row < end; row += paged::kMergeThreads / CH) {
      const int r_in = row & 127;
      const int in_tile = static_cast<int>((static_cast<float>(r_in) + 0.5f) * inv);  // r_in / G, exact below 128
      const int tok = (row >> 7) * tpt + in_tile;                                      // of the pair's tokens
      if (r_in >= tpt * p.G || tok >= it.y) continue;
      float m = -INFINITY, l = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      paged::join_pieces<4>(p.tc_o + c, p.tc_ml, (slot - mine) * kRowsOfItem + row, kRowsOfItem, pieces, DV, m, l, acc);
      paged::store_row<__half>(p, static_cast<int64_t>(it.x + tok) * p.H_q + it.z * p.G + r_in - in_tile * p.G, c, acc, m, l);
    }
  }
}


}  // namespace paged_tc
}  // namespace sdpa_b200
