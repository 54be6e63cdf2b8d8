// Translation unit: head norms with rotation (forward, backward, cache write)
#include "host.cuh"
#include "rotary.cuh"

#include <algorithm>

using namespace sdpa_b200;
using namespace sdpa_b200::host;

namespace {

// Lanes a head row takes (eight features each): a power of two for the shuffles.
int lanes_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : 16; }

// Shares of a token's head groups: enough of them that short inputs still
// fill the device (two rounds of 2048 threads an SM), one when there are
// tokens enough (a share reads its token's position and table row again).
int shares(int64_t tokens, int lanes, int units) {
  const int64_t have = tokens * lanes, want = static_cast<int64_t>(num_sms()) * 4096;
  return static_cast<int>(std::min<int64_t>(units, std::max<int64_t>(1, (want + have - 1) / have)));
}

int units_of(int heads) { return (heads + rotary::kHeads - 1) / rotary::kHeads; }

template <typename Kernel>
int launch_grid(Kernel kern, int64_t gx, int gy, int threads, cudaStream_t st, const rotary::Params& p, int* launches) {
  if (gx <= 0 || gx > 0x7fffffffLL || gy > 65535) return SDPA_B200_EINVAL;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
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

template <typename T, int LANES>
int forward_t(const rotary::Params& p, cudaStream_t st, int* launches) {
  constexpr int kGroups = rotary::kThreads / LANES;
  const int64_t tokens = std::max(p.q.tokens, p.k.tokens);
  const int units = units_of(p.q.heads) + units_of(p.k.heads);
  return launch_grid(rotary::forward_kernel<T, LANES>, (tokens + kGroups - 1) / kGroups, shares(tokens, LANES, units),
                     rotary::kThreads, st, p, launches);
}

template <typename T, int LANES>
int append_t(const rotary::Params& p, cudaStream_t st, int* launches) {
  constexpr int kGroups = rotary::kThreads / LANES;
  const int nv = p.k.heads * p.D_v / static_cast<int>(16 / sizeof(T));
  const int units = units_of(p.q.heads) + units_of(p.k.heads) + (nv + LANES * rotary::kHeads - 1) / (LANES * rotary::kHeads);
  return launch_grid(rotary::append_kernel<T, LANES>, (p.view.tokens + kGroups - 1) / kGroups,
                     shares(p.view.tokens, LANES, units), rotary::kThreads, st, p, launches);
}

template <typename T, int LANES>
int backward_t(rotary::Params p, cudaStream_t st, int* launches) {
  constexpr int kGroups = rotary::kThreads / LANES;
  const int64_t tokens = std::max(p.q.tokens, p.k.tokens);
  // one block at least: without tokens the weights' gradients are zeros
  p.blocks = static_cast<int>(std::min<int64_t>(rotary::kGradBlocks, std::max<int64_t>(1, (tokens + kGroups - 1) / kGroups)));
  if (int r = launch_grid(rotary::backward_kernel<T, LANES>, p.blocks, 1, rotary::kThreads, st, p, launches)) return r;
  if (!p.dw_q && !p.dw_k) return SDPA_B200_OK;
  return launch_grid(rotary::weight_kernel<T>, (p.D + 31) / 32, 2, 1024, st, p, launches);
}

template <typename T>
int dispatch(const rotary::Params& p, int what, cudaStream_t st, int* launches) {
  const int lanes = lanes_of(p.D);
  if (what == 0)
    return lanes == 4   ? forward_t<T, 4>(p, st, launches)
           : lanes == 8 ? forward_t<T, 8>(p, st, launches)
                        : forward_t<T, 16>(p, st, launches);
  if (what == 1)
    return lanes == 4   ? append_t<T, 4>(p, st, launches)
           : lanes == 8 ? append_t<T, 8>(p, st, launches)
                        : append_t<T, 16>(p, st, launches);
  return lanes == 4   ? backward_t<T, 4>(p, st, launches)
         : lanes == 8 ? backward_t<T, 8>(p, st, launches)
                      : backward_t<T, 16>(p, st, launches);
}

int by_type(int dtype, const rotary::Params& p, int what, cudaStream_t st, int* launches) {
  return dtype == SDPA_B200_F16 ? dispatch<__half>(p, what, st, launches) : dispatch<float>(p, what, st, launches);
}

}  // namespace

int sdpa_b200::launch_rotary_fwd(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, 0, st, launches);
}
int sdpa_b200::launch_paged_append(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, 1, st, launches);
}
int sdpa_b200::launch_rotary_bwd(int dtype, const rotary::Params& p, cudaStream_t st, int* launches) {
  return by_type(dtype, p, 2, st, launches);
}

SDPA_B200_STATUS_EXCHANGE(rotary)
