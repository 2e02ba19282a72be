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
  switch (l.nt) {
    case 16: return launch<MODE, ACT, 16>(m, p, l, s);
    case 32: return launch<MODE, ACT, 32>(m, p, l, s);
    default: return launch<MODE, ACT, 64>(m, p, l, s);
  }
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
  // The time of a split: the bytes that the busiest SM takes in, at the 85-100 B/ns that a SM
  // takes from L2, and the exchange of the sums (two cluster barriers, then about 15 B/ns).
  // Measured, 1 x 1024 x 4096: 30.8, 20.9, 15.0, 13.7 us for 1, 2, 4, 8 CTAs a tile; 24 x 4096 x
  // 16384: 127, 95, 88, 93 us.
  const int products = mode == FEW_GATED ? 2 : 1;
  FewPlan best{};
  best.nt = columns <= 16 ? 16 : columns <= 32 ? 32 : 64;
  best.tiles = static_cast<int>((F + 127) / 128);
  double best_ns = 0;
  for (int q = 1; q <= 8 && q <= kb; q *= 2) {
    const long long turns = (static_cast<long long>(best.tiles) * q + sms - 1) / sms;
    const double bytes = static_cast<double>((kb + q - 1) / q) * (products * 16384 + best.nt * 128);
    const double ns = turns * bytes / 100.0 + (q > 1 ? 1200.0 + best.nt * products * 512.0 * (q - 1) / q / 15.0 : 0.0);
    if (q == 1 || ns < best_ns) best.q = q, best_ns = ns;
  }
  return best;
}

cudaError_t launch_few(int mode, int act, const FewMaps& m, const FewParams& p, const FewPlan& plan, cudaStream_t stream) {
  if (mode == FEW_GATED) return by_act<FEW_GATED>(act, m, p, plan, stream);
  if (mode == FEW_DGATE) return by_act<FEW_DGATE>(act, m, p, plan, stream);
  return by_tokens<FEW_PLAIN, ACT_NONE>(m, p, plan, stream);
}

}  // namespace fo
