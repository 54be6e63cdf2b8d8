// Translation unit: attention over the paged cache, the kernels for few rows
// and the choice between them and paged_tc.cu's for chunks
#include "host.cuh"
#include "paged_mma.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

int bucket_of(int D, int D_v) { return std::max(D, D_v) <= 64 ? 64 : 128; }

// Row tiles of 16 a CTA takes together, from the mean number of packed rows
// (new tokens x heads of a group) of a sequence: the rows of one CTA share one
// reading of the keys.
int row_tiles_of(int64_t tokens, int64_t seqs, int64_t group) {
  const int64_t mean = (tokens * group + seqs - 1) / std::max<int64_t>(seqs, 1);
  return mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
}

// Workspace of the cut items: [ranges][2][rows] sums, (max, sum) pairs, one record a range.
struct Layout {
  size_t o, ml, item, bytes;
};
template <typename T, int DB, int MT>
Layout layout_of() {
  using S = paged::Shape<T, DB, MT>;
  const size_t ranges = static_cast<size_t>(S::kCtas) * num_sms() * S::kGroups;
  const size_t n = ranges * 2 * S::kRowsAll;
  Layout l;
  l.o = 0;
  l.ml = l.o + n * DB * sizeof(float);
  l.item = l.ml + n * sizeof(float2);
  l.bytes = l.item + ranges * sizeof(int4);
  return l;
}

template <typename T, int DB, int MT>
int launch_mma_t(paged::Params p, void* workspace, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> attr_done{0};
  using S = paged::Shape<T, DB, MT>;
  auto kern = paged::attend_kernel<T, DB, MT>;
  if (cudaError_t e = ensure_smem(kern, S::kSmemBytes, attr_done)) return cuda_failure("shared-memory attribute", e);
  const int ctas = S::kCtas * num_sms();
  const Layout l = layout_of<T, DB, MT>();
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(w + l.o);
  p.part_ml = reinterpret_cast<float2*>(w + l.ml);
  p.part_item = reinterpret_cast<int4*>(w + l.item);
  CUtensorMap mk, mv;
  const int64_t page = int64_t(1) << p.view.page_shift;
  if (!make_pool_map(&mk, sizeof(T), p.k_pages, p.view.num_pages, page, p.H_kv, p.D, S::kKeys) ||
      !make_pool_map(&mv, sizeof(T), p.v_pages, p.view.num_pages, page, p.H_kv, p.D_v, S::kKeys))
    return SDPA_B200_ECUDA;  // detail recorded by make_map_4d
  if (int r = launch_tc(kern, ctas, paged::kThreads, S::kSmemBytes, st, mk, mv, p)) return r;
  ++*launches;
  if (int r = launch_tc(paged::merge_kernel<T, DB, MT>, ctas * S::kGroups, paged::kMergeThreads, 0, st, p)) return r;
  ++*launches;
  return SDPA_B200_OK;
}

template <typename T, int DB>
int launch_mma(const paged::Params& p, void* ws, int mt, cudaStream_t st, int* launches) {
  return mt == 1   ? launch_mma_t<T, DB, 1>(p, ws, st, launches)
         : mt == 2 ? launch_mma_t<T, DB, 2>(p, ws, st, launches)
                   : launch_mma_t<T, DB, 4>(p, ws, st, launches);
}

template <typename T, int DB>
size_t bytes_of(int mt) {
  return mt == 1 ? layout_of<T, DB, 1>().bytes : mt == 2 ? layout_of<T, DB, 2>().bytes : layout_of<T, DB, 4>().bytes;
}

}  // namespace

// Chunks go to the tcgen05 kernel: fp16, a head group that fits its 128-row
// tiles, and more than one 16-row tile of packed rows a sequence on average
// (the lengths themselves are on the device).
static bool use_tc(int dtype, int64_t tokens, int64_t seqs, int64_t group) {
  return dtype == SDPA_B200_F16 && group <= 128 && tokens * group > 16 * seqs;
}

size_t sdpa_b200::paged_workspace_bytes(int dtype, int64_t tokens, int64_t seqs, int64_t H_q, int64_t H_kv, int64_t D,
                                        int64_t D_v) {
  if (use_tc(dtype, tokens, seqs, H_q / H_kv)) return paged_tc_workspace_bytes(static_cast<int>(D_v));
  const int mt = row_tiles_of(tokens, seqs, H_q / H_kv);
  const bool small = bucket_of(static_cast<int>(D), static_cast<int>(D_v)) == 64;
  if (dtype == SDPA_B200_F16) return small ? bytes_of<__half, 64>(mt) : bytes_of<__half, 128>(mt);
  return small ? bytes_of<float, 64>(mt) : bytes_of<float, 128>(mt);
}

int sdpa_b200::launch_paged_sdpa(int dtype, paged::Params p, void* workspace, cudaStream_t st, int* launches) {
  const int mt = row_tiles_of(p.view.tokens, p.view.seqs, p.G);
  p.sms = num_sms();
  if (use_tc(dtype, p.view.tokens, p.view.seqs, p.G)) return launch_paged_tc(p, workspace, st, launches);
  const bool small = bucket_of(p.D, p.D_v) == 64;
  if (dtype == SDPA_B200_F16)
    return small ? launch_mma<__half, 64>(p, workspace, mt, st, launches) : launch_mma<__half, 128>(p, workspace, mt, st, launches);
  return small ? launch_mma<float, 64>(p, workspace, mt, st, launches) : launch_mma<float, 128>(p, workspace, mt, st, launches);
}

SDPA_B200_STATUS_EXCHANGE(paged)
