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

int max_ctas() { return 2 * num_sms(); }

// Workspace of the cut items: [ctas][2][rows] sums, (max, sum) pairs, one record a CTA.
struct Layout {
  size_t o, ml, item, bytes;
};
Layout layout_of(int ctas, int rows, int db) {
  const size_t n = static_cast<size_t>(ctas) * 2 * rows;
  Layout l;
  l.o = 0;
  l.ml = l.o + n * db * sizeof(float);
  l.item = l.ml + n * sizeof(float2);
  l.bytes = l.item + static_cast<size_t>(ctas) * sizeof(int4);
  return l;
}

template <typename T, int DB, int MT>
int launch_mma_t(paged::Params p, void* workspace, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> attr_done{0};
  auto kern = paged::attend_kernel<T, DB, MT>;
  const size_t smem = sizeof(paged::Smem<DB, MT>) + (sizeof(T) == 4 ? static_cast<size_t>(MT) * (DB / 16) * 4 * 32 * 16 : 0);
  if (cudaError_t e = ensure_smem(kern, smem, attr_done)) return cuda_failure("shared-memory attribute", e);
  const int ctas = max_ctas();
  const Layout l = layout_of(ctas, paged::kRows * MT, DB);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(w + l.o);
  p.part_ml = reinterpret_cast<float2*>(w + l.ml);
  p.part_item = reinterpret_cast<int4*>(w + l.item);
  if (int r = launch_tc(kern, ctas, paged::kThreads, smem, st, p)) return r;
  ++*launches;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), paged::kRows * MT * (DB / 4) / paged::kThreads);
  cfg.blockDim = dim3(paged::kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged::merge_kernel<T, DB, MT>, p);
  if (e != cudaSuccess) return cuda_failure("kernel launch", e);
  ++*launches;
  return SDPA_B200_OK;
}

template <typename T, int DB>
int launch_mma(const paged::Params& p, void* ws, int mt, cudaStream_t st, int* launches) {
  return mt == 1   ? launch_mma_t<T, DB, 1>(p, ws, st, launches)
         : mt == 2 ? launch_mma_t<T, DB, 2>(p, ws, st, launches)
                   : launch_mma_t<T, DB, 4>(p, ws, st, launches);
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
  return layout_of(max_ctas(), paged::kRows * mt, bucket_of(static_cast<int>(D), static_cast<int>(D_v))).bytes;
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
