// fo_few.cu -- instantiations, work split and launch of the short-token products.
#include "fo_few.cuh"
#include "fo_host.cuh"
#include "../../include/b200fo.h"

namespace fo {
namespace {

template <int MODE, int ACT, int NT>
cudaError_t launch(const FewMaps& m, const FewParams& p, const FewPlan& l, cudaStream_t s) {
  static std::atomic<uint64_t> opted{0};
  return launch_pdl(fo_few_kernel<MODE, ACT, NT>, opted, dim3(l.tiles * l.q), dim3(kFewThreads), FewShape<MODE, NT>::kSmem, l.q, s, m, p);
}

template <int MODE, int ACT>
cudaError_t by_tokens(const FewMaps& m, const FewParams& p, const FewPlan& l, cudaStream_t s) {
  if (l.nt == 16) return launch<MODE, ACT, 16>(m, p, l, s);
  if constexpr (MODE != FEW_GATED) {  // which has one column a token, 32 at most
    if (l.nt == 64) return launch<MODE, ACT, 64>(m, p, l, s);
  }
  return launch<MODE, ACT, 32>(m, p, l, s);
}

template <int MODE>
cudaError_t by_act(int act, const FewMaps& m, const FewParams& p, const FewPlan& l, cudaStream_t s) {
  switch (act) {
    case FO_GATE_SILU: return by_tokens<MODE, ACT_SILU>(m, p, l, s);
    case FO_GATE_GELU_TANH: return by_tokens<MODE, ACT_GELU_TANH>(m, p, l, s);
    case FO_GATE_GELU_ERF: return by_tokens<MODE, ACT_GELU_ERF>(m, p, l, s);
    default: return by_tokens<MODE, ACT_RELU>(m, p, l, s);
  }
}

}  // namespace

FewPlan few_plan(int mode, int64_t F, int64_t columns, int kb, int sms) {
  // As many CTAs as are resident at once, two a SM: one CTA keeps 110 KB under way, 43 B/ns of
  // HBM; but K blocks enough that the exchange of the sums stays small beside them.  Measured,
  // blocks with the gated product in 1, 2, 4, 8 CTAs a tile: 1 x 4096 x 16384 (128 tiles) 71, 67,
  // 71, 74 us; 24 tokens 84, 79, 85, 92; 8 x 2048 x 8192 (64 tiles) 33, 31, 28, 34; 1 x 1024 x
  // 4096 (32 tiles, 16 K blocks) 15.1, 13.0, 11.7, 11.7.  With the second product so (32 tiles),
  // 1 x 4096 x 16384: 120, 85, 73, 67; backward, 64 x 1024 x 4096: 111, 88, 62, 50.
  const int products = mode == FEW_GATED ? 2 : 1;
  FewPlan best{};
  best.nt = columns <= 16 ? 16 : columns <= 32 ? 32 : 64;
  best.tiles = static_cast<int>((F + 127) / 128);
  best.q = 1;
  while (best.q < 8 && 2ll * best.tiles * best.q <= 2 * sms && 4 * products * best.q <= kb) best.q *= 2;
  return best;
}

cudaError_t launch_few(int mode, int act, const FewMaps& m, const FewParams& p, const FewPlan& plan, cudaStream_t stream) {
  if (mode == FEW_GATED) return by_act<FEW_GATED>(act, m, p, plan, stream);
  if (mode == FEW_DGATE) return by_act<FEW_DGATE>(act, m, p, plan, stream);
  return by_tokens<FEW_PLAIN, ACT_NONE>(m, p, plan, stream);
}

}  // namespace fo
