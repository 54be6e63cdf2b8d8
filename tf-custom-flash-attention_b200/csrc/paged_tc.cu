// Translation unit: attention of chunks over the paged cache (tcgen05)
#include "host.cuh"
#include "paged_tc.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

// Pieces of cut items: at most one an SM and one an item (fewer items than SMs).
int max_slots() { return 2 * num_sms(); }
int v_bucket(int D_v) { return D_v <= 64 ? 64 : 128; }

bool map_4d(CUtensorMap* m, const void* base, const int64_t (&dims)[4], const int64_t (&strides)[3], const int (&box)[4]) {
  auto fn = encode_fn();
  if (!fn) return map_failure(0, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], e[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) d[i] = static_cast<cuuint64_t>(dims[i]), b[i] = static_cast<cuuint32_t>(box[i]);
  for (int i = 0; i < 3; ++i) s[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), d, s, b, e,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS || map_failure(static_cast<int>(r), "cuTensorMapEncodeTiled");
}

// Pool [pages, page, H_kv, D]: boxes of one 128-byte row segment x 1 head x min(page, 128) rows x 1 page.
bool pool_map(CUtensorMap* m, const void* base, const paged::Params& p, int D) {
  const int64_t page = int64_t(1) << p.view.page_shift;
  return map_4d(m, base, {D, p.H_kv, page, p.view.num_pages}, {D, int64_t(p.H_kv) * D, page * p.H_kv * D},
                {64, 1, static_cast<int>(std::min<int64_t>(page, tc::kBN)), 1});
}

template <int DQK, int DV>
int launch_t(paged::Params p, void* workspace, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> attr_done{0};
  using C = paged_tc::Cfg<DQK, DV>;
  auto kern = paged_tc::attend_kernel<DQK, DV>;
  if (cudaError_t e = ensure_smem(kern, C::kSmemBytes, attr_done)) return cuda_failure("shared-memory attribute", e);
  const int tpt = tc::kBM / p.G;  // tokens of a row tile
  CUtensorMap mq, mk, mv;
  if (!map_4d(&mq, p.q, {p.D, p.G, p.H_kv, p.view.tokens}, {p.D, int64_t(p.G) * p.D, p.q_stride}, {64, p.G, 1, tpt}) ||
      !pool_map(&mk, p.k_pages, p, p.D) || !pool_map(&mv, p.v_pages, p, p.D_v))
    return SDPA_B200_ECUDA;  // detail recorded by map_4d
  const int64_t rows = static_cast<int64_t>(max_slots()) * 2 * tc::kBM;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * DV);
  // items of N sequences: at most T / (tokens a pair) + N a KV head; pieces beyond the items: at most one an SM
  const int64_t items = (p.view.tokens / (2 * tpt) + static_cast<int64_t>(p.view.seqs)) * p.H_kv;
  if (int r = launch_tc(kern, items + p.sms, paged_tc::kThreads, C::kSmemBytes, st, mq, mk, mv, p)) return r;
  ++*launches;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(max_slots()), 8);
  cfg.blockDim = dim3(paged_tc::kMergeThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_tc::merge_kernel<DV>, p);
  if (e != cudaSuccess) return cuda_failure("kernel launch", e);
  ++*launches;
  return SDPA_B200_OK;
}

}  // namespace

size_t sdpa_b200::paged_tc_workspace_bytes(int D_v) {
  return static_cast<size_t>(max_slots()) * 2 * tc::kBM * (v_bucket(D_v) * sizeof(float) + sizeof(float2));
}

int sdpa_b200::launch_paged_tc(const paged::Params& p, void* workspace, cudaStream_t st, int* launches) {
  if (p.D > 64)
    return p.D_v > 64 ? launch_t<128, 128>(p, workspace, st, launches) : launch_t<128, 64>(p, workspace, st, launches);
  return p.D_v > 64 ? launch_t<64, 128>(p, workspace, st, launches) : launch_t<64, 64>(p, workspace, st, launches);
}

SDPA_B200_STATUS_EXCHANGE(paged_tc)
