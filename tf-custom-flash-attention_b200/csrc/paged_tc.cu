// Translation unit: attention of chunks over the paged cache (tcgen05)
#include "host.cuh"
#include "paged_tc.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

// Pieces of a call: with at least as many items as SMs at most one an SM; with
// fewer, an item has at most 4/3 of its cost in quanta (5/4 of the SMs' in all),
// or one: at most 5/3 + 1 an SM.
int max_slots() { return 3 * num_sms(); }
int v_bucket(int D_v) { return D_v <= 64 ? 64 : 128; }

template <int DQK, int DV>
int launch_t(const paged::Params& p, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> attr_done{0};
  using C = paged_tc::Cfg<DQK, DV>;
  auto kern = paged_tc::attend_kernel<DQK, DV>;
  if (cudaError_t e = ensure_smem(kern, C::kSmemBytes, attr_done)) return cuda_failure("shared-memory attribute", e);
  const int tpt = tc::kBM / p.G;  // tokens of a row tile
  CUtensorMap mq, mk, mv;
  const int64_t page = int64_t(1) << p.view.page_shift;
  const int box = static_cast<int>(std::min<int64_t>(page, paged_tc::kBN));
  if (!make_map_4d(&mq, 2, p.q, {p.D, p.G, p.H_kv, p.view.tokens}, {p.D, int64_t(p.G) * p.D, p.q_stride}, {64, p.G, 1, tpt}) ||
      !make_pool_map(&mk, 2, p.k_pages, p.view.num_pages, page, p.H_kv, p.D, box) ||
      !make_pool_map(&mv, 2, p.v_pages, p.view.num_pages, page, p.H_kv, p.D_v, box))
    return SDPA_B200_ECUDA;  // detail recorded by make_map_4d
  // items of N sequences: at most T / (tokens a pair) + N a KV head; pieces beyond one an item: at most 5/4 an SM
  const int64_t items = (p.view.tokens / (2 * tpt) + static_cast<int64_t>(p.view.seqs)) * p.H_kv;
  if (int r = launch_tc(kern, items + 5 * p.sms / 4, paged_tc::kThreads, C::kSmemBytes, st, mq, mk, mv, p)) return r;
  ++*launches;
  if (int r = launch_tc(paged_tc::merge_kernel<DV>, 4 * p.sms, paged::kMergeThreads, 0, st, p)) return r;
  ++*launches;
  return SDPA_B200_OK;
}

}  // namespace

// Places the chunk kernel's workspace at w (p null: only its bytes).
size_t sdpa_b200::place_paged_tc(paged::Params* p, void* w, int D_v) {
  const size_t slots = static_cast<size_t>(max_slots()), rows = slots * 2 * tc::kBM, cols = v_bucket(D_v);
  if (p) {
    p->tc_o = static_cast<float*>(w);
    p->tc_ml = reinterpret_cast<float2*>(p->tc_o + rows * cols);
    p->tc_item = reinterpret_cast<int4*>(p->tc_ml + rows);
    p->tc_slots = reinterpret_cast<int*>(p->tc_item + slots);
  }
  return rows * (cols * sizeof(float) + sizeof(float2)) + slots * sizeof(int4) + 16;
}

int sdpa_b200::launch_paged_tc(const paged::Params& p, cudaStream_t st, int* launches) {
  if (p.D > 64)
    return p.D_v > 64 ? launch_t<128, 128>(p, st, launches) : launch_t<128, 64>(p, st, launches);
  return p.D_v > 64 ? launch_t<64, 128>(p, st, launches) : launch_t<64, 64>(p, st, launches);
}

SDPA_B200_STATUS_EXCHANGE(paged_tc)
