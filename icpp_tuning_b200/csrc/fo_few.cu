#include <cstdlib>
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
    case 64: return launch<MODE, ACT, 64>(m, p, l, s);
    case 128: return launch<MODE, ACT, 128>(m, p, l, s);
    case 256:
      if constexpr (MODE != FEW_GATED) return launch<MODE, ACT, 256>(m, p, l, s);
  }
  return cudaErrorInvalidValue;
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

FewPlan few_plan(int mode, int64_t F, int64_t T, int kb, int sms) {
  // The time of a choice: the bytes the busiest SM takes in, at about 100 B/ns, and for a
  // split the exchange of the sums.
  const int products = mode == FEW_GATED ? 2 : 1;
  FewPlan best{};
  double best_ns = 0;
  static const int env_nt = getenv("FO_NT") ? atoi(getenv("FO_NT")) : 0, env_q = getenv("FO_Q") ? atoi(getenv("FO_Q")) : 0;
  for (int nt = 16; nt <= (mode == FEW_GATED ? 128 : 256); nt *= 2) {
    const int tok_tiles = static_cast<int>((T + nt - 1) / nt);
    const long long tiles = (F + 127) / 128 * tok_tiles;
    for (int q = 1; q <= 8 && q <= kb; q *= 2) {
      const long long ctas = tiles * q;
      const long long turns = (ctas + sms - 1) / sms;
      const double bytes = static_cast<double>((kb + q - 1) / q) * (products * 16384 + nt * 128);
      const double ns = turns * bytes / 100.0 + (q > 1 ? 1200.0 + nt * products * 512.0 * (q - 1) / q / 15.0 : 0.0);
      if ((env_nt && nt != env_nt) || (env_q && q != env_q)) continue;
      if (best.nt == 0 || ns < best_ns) best = {nt, tok_tiles, static_cast<int>(tiles), q}, best_ns = ns;
    }
  }
  return best;
}

cudaError_t launch_few(int mode, int act, const FewMaps& m, FewParams p, const FewPlan& plan, cudaStream_t stream) {
  p.tok_tiles = plan.tok_tiles;
  if (mode == FEW_GATED) return by_act<FEW_GATED>(act, m, p, plan, stream);
  if (mode == FEW_DGATE) return by_act<FEW_DGATE>(act, m, p, plan, stream);
  return by_tokens<FEW_PLAIN, ACT_NONE>(m, p, plan, stream);
}

}  // namespace fo
