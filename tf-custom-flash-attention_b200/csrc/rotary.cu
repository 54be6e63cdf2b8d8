// Translation unit: head norms with rotation (forward, backward, cache write)
#include "host.cuh"
#include "rotary.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

// Shares of a token's head groups: enough of them that short inputs still
// fill the device (two rounds of 2048 threads an SM), one when there are
// tokens enough (a share reads its token's position and table row again).
int shares(int64_t tokens, int lanes, int units) {
  const int64_t have = tokens * lanes, want = static_cast<int64_t>(num_sms()) * 4096;
  return static_cast<int>(std::min<int64_t>(units, std::max<int64_t>(1, (want + have - 1) / have)));
}

template <typename Kernel>
int launch_grid(Kernel kern, int64_t gx, int gy, int threads, size_t smem, cudaStream_t st, const rotary::Params& p,
                int* launches) {
  if (gx <= 0 || gx > 0x7fffffffLL || gy > 65535) return SDPA_B200_EINVAL;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return cuda_failure("kernel launch", e);
  ++*launches;
  return SDPA_B200_OK;
}

enum { kForward, kAppend, kBackward };

template <typename T, int LANES, bool INTER>
int launch_t(rotary::Params p, int what, cudaStream_t st, int* launches) {
  constexpr int kGroups = rotary::kThreads / LANES, N = rotary::kHeadsAhead;
  if (what == kBackward) {
    const int64_t tokens = std::max(p.q.tokens, p.k.tokens);
    // One wave, two blocks an SM: more of them start their ring and write their sums again (32768 tokens x 40 heads x 128
    // fp16: 184 us, 187 with twice the blocks, 193 with four times; 4099 x 32 x 64 fp32: 21 and 25).  One block at
    // least: without tokens the weights' gradients are zeros.
    const int64_t most = std::min(rotary::kGradBlocks, 2 * num_sms());
    const int64_t gx = std::min<int64_t>(most, std::max<int64_t>(1, (tokens + kGroups - 1) / kGroups));
    const int gy = static_cast<int>(std::min<int64_t>(std::max({1, p.q.heads / 4, p.k.heads / 4}), most / gx));
    p.blocks = static_cast<int>(gx) * gy;
    static std::atomic<uint64_t> attr_done{0};
    constexpr size_t kRing = rotary::kStages<T> * rotary::kStageBytes<T>;
    auto kern = rotary::backward_kernel<T, LANES, INTER>;
    if (cudaError_t e = ensure_smem(kern, kRing, attr_done)) return cuda_failure("shared-memory attribute", e);
    if (int r = launch_grid(kern, gx, gy, rotary::kThreads, kRing, st, p, launches)) return r;
    if (!p.dw_q && !p.dw_k) return SDPA_B200_OK;
    return launch_grid(rotary::weight_kernel<T>, (p.D + 31) / 32, 2, 1024, 0, st, p, launches);
  }
  const int heads = rotary::units_of(p.q.heads, N) + rotary::units_of(p.k.heads, N);
  if (what == kForward) {
    const int64_t tokens = std::max(p.q.tokens, p.k.tokens);
    return launch_grid(rotary::forward_kernel<T, LANES, INTER>, (tokens + kGroups - 1) / kGroups,
                       shares(tokens, LANES, heads), rotary::kThreads, 0, st, p, launches);
  }
  const int nv = p.k.heads * p.D_v / static_cast<int>(16 / sizeof(T));
  return launch_grid(rotary::append_kernel<T, LANES, INTER>, (p.view.tokens + kGroups - 1) / kGroups,
                     shares(p.view.tokens, LANES, heads + rotary::units_of(nv, LANES * rotary::kCopyWords)), rotary::kThreads,
                     0, st, p, launches);
}

// Eight features a lane, a power of two of lanes a head row.
template <typename T>
int dispatch(rotary::Params p, int what, cudaStream_t st, int* launches) {
  p.inv_D = 1.0f / static_cast<float>(p.D);
  const bool inter = p.interleaved != 0;
  if (p.D > 64) return inter ? launch_t<T, 16, true>(p, what, st, launches) : launch_t<T, 16, false>(p, what, st, launches);
  return inter ? launch_t<T, 8, true>(p, what, st, launches) : launch_t<T, 8, false>(p, what, st, launches);
}

int by_type(int dtype, const rotary::Params& p, int what, cudaStream_t st, int* launches) {
  return dtype == SDPA_B200_F16 ? dispatch<__half>(p, what, st, launches) : dispatch<float>(p, what, st, launches);
}

}  // namespace

int sdpa_b200::launch_rotary_fwd(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, kForward, st, launches);
}
int sdpa_b200::launch_paged_append(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, kAppend, st, launches);
}
int sdpa_b200::launch_rotary_bwd(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, kBackward, st, launches);
}

SDPA_B200_STATUS_EXCHANGE(rotary)
