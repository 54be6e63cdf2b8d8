// Translation unit: attention over the paged cache, the kernels for few rows,
// the merge, and the choice between them and paged_tc.cu's for chunks
#include "host.cuh"
#include "paged_mma.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

int bucket_of(int64_t D, int64_t D_v) { return std::max(D, D_v) <= 64 ? 64 : 128; }

// The kernel a call takes.  The lengths are on the device, so the rule goes by
// the call's tokens and sequences alone.  fp16: the few-row kernel for at most a
// token a sequence, or so few more that none has over 16 packed rows (new tokens x
// heads of a group) even if one has them all; the tcgen05 kernel for the rest with
// groups of up to 128 heads, what its row tiles hold.  (The bound knows no single
// sequence's tokens: drafts of a few tokens each in many sequences go to the
// tcgen05 kernel though their rows are few, and a chunk among as many sequences
// without new tokens to the few-row one, where it is right but slow.)  It serves
// single tokens among chunks as well (few-row and tcgen05 kernel, us: 16 x 32768
// keys x 4 heads 181 and 178; 32 ragged to 8192 keys x 8 heads 57 and 90; 64 x 1000
// keys, 8 / 16 / 32 rows, 58 / 63 / 84 and 75 / 77 / 79; one token of 32 heads to a
// KV head, 8 x 4096 keys, 62 and 18), while a chunk in the few-row kernel reads its
// keys once every 16 rows.
// fp32: the few-row kernel, its row tiles from the mean of packed rows: a thin
// tile of 8 a warp up to two of them (16 x 8192 keys x 2 heads x 128, 16 rows: 99 us
// against 127 with tiles of 16 in pairs; 16 x 2000 keys x 4 heads, 12 rows: 57 and 73),
// then two and four tiles of 16 that share a ring.
struct Plan {
  bool tc;
  int mt;  // row tiles of a group of warps
};
Plan plan_of(int dtype, int64_t tokens, int64_t seqs, int64_t group) {
  if (dtype == SDPA_B200_F16 && group <= 128) return {group > 16 || (tokens > seqs && (tokens - seqs + 1) * group > 16), 1};
  if (dtype == SDPA_B200_F16) return {false, 4};  // over 128 rows a token
  const int64_t mean = (tokens * group + seqs - 1) / seqs;
  return {false, mean <= 16 ? 1 : mean <= 32 ? 2 : 4};
}

// Workspace of the few-row kernel: [ranges][2][rows] sums, (max, sum) pairs, one record a range.
template <typename T, int DB, int MT>
size_t place_mma_t(paged::Params* p, uint8_t* w) {
  using S = paged::Shape<T, DB, MT>;
  const int ranges = S::kCtas * num_sms() * S::kGroups;
  const size_t n = static_cast<size_t>(ranges) * 2 * S::kRowsAll;
  if (p) {
    p->part_o = reinterpret_cast<float*>(w);
    p->part_ml = reinterpret_cast<float2*>(w + n * DB * sizeof(float));
    p->part_item = reinterpret_cast<int4*>(w + n * (DB * sizeof(float) + sizeof(float2)));
    p->part_ranges = ranges;
    p->part_rows = S::kRowsAll;
    p->part_cols = DB;
  }
  return n * (DB * sizeof(float) + sizeof(float2)) + ranges * sizeof(int4);
}

template <typename T, int DB, int MT>
int launch_mma_t(const paged::Params& p, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> attr_done{0};
  using S = paged::Shape<T, DB, MT>;
  auto kern = paged::attend_kernel<T, DB, MT>;
  if (cudaError_t e = ensure_smem(kern, S::kSmemBytes, attr_done)) return cuda_failure("shared-memory attribute", e);
  CUtensorMap mk, mv;
  const int64_t page = int64_t(1) << p.view.page_shift;
  if (!make_pool_map(&mk, sizeof(T), p.k_pages, p.view.num_pages, page, p.H_kv, p.D, S::kKeys) ||
      !make_pool_map(&mv, sizeof(T), p.v_pages, p.view.num_pages, page, p.H_kv, p.D_v, S::kKeys))
    return SDPA_B200_ECUDA;  // detail recorded by make_map_4d
  if (int r = launch_tc(kern, S::kCtas * num_sms(), paged::kThreads, S::kSmemBytes, st, mk, mv, p)) return r;
  ++*launches;
  return SDPA_B200_OK;
}

// F<T, DB, MT>(args) for the call's type, bucket and row tiles (fp16: 1 or 4).
#define SDPA_B200_PAGED_DISPATCH(F, dtype, db, mt, ...)                                                   \
  ((dtype) == SDPA_B200_F16                                                                               \
       ? ((db) == 64 ? ((mt) == 1 ? F<__half, 64, 1>(__VA_ARGS__) : F<__half, 64, 4>(__VA_ARGS__))        \
                     : ((mt) == 1 ? F<__half, 128, 1>(__VA_ARGS__) : F<__half, 128, 4>(__VA_ARGS__)))     \
       : ((db) == 64 ? ((mt) == 1   ? F<float, 64, 1>(__VA_ARGS__)                                        \
                        : (mt) == 2 ? F<float, 64, 2>(__VA_ARGS__)                                        \
                                    : F<float, 64, 4>(__VA_ARGS__))                                       \
                     : ((mt) == 1   ? F<float, 128, 1>(__VA_ARGS__)                                       \
                        : (mt) == 2 ? F<float, 128, 2>(__VA_ARGS__)                                       \
                                    : F<float, 128, 4>(__VA_ARGS__))))

size_t place_mma(const Plan& plan, int dtype, int db, paged::Params* p, uint8_t* w) {
  return SDPA_B200_PAGED_DISPATCH(place_mma_t, dtype, db, plan.mt, p, w);
}

}  // namespace

size_t sdpa_b200::paged_workspace_bytes(int dtype, int64_t tokens, int64_t seqs, int64_t H_q, int64_t H_kv, int64_t D,
                                        int64_t D_v) {
  const Plan plan = plan_of(dtype, tokens, seqs, H_q / H_kv);
  return plan.tc ? place_paged_tc(nullptr, nullptr, static_cast<int>(D_v))
                 : place_mma(plan, dtype, bucket_of(D, D_v), nullptr, nullptr);
}

int sdpa_b200::launch_paged_sdpa(int dtype, paged::Params p, void* workspace, cudaStream_t st, int* launches) {
  const Plan plan = plan_of(dtype, p.view.tokens, p.view.seqs, p.G);
  const int db = bucket_of(p.D, p.D_v);
  p.sms = num_sms();
  if (plan.tc) {
    place_paged_tc(&p, workspace, p.D_v);
    return launch_paged_tc(p, st, launches);
  }
  place_mma(plan, dtype, db, &p, static_cast<uint8_t*>(workspace));
  if (int r = SDPA_B200_PAGED_DISPATCH(launch_mma_t, dtype, db, plan.mt, p, st, launches)) return r;
  auto merge = dtype == SDPA_B200_F16 ? paged::merge_kernel<__half> : paged::merge_kernel<float>;
  if (int r = launch_tc(merge, 8 * p.sms, paged::kMergeThreads, 0, st, p)) return r;
  ++*launches;
  return SDPA_B200_OK;
}

SDPA_B200_STATUS_EXCHANGE(paged)
