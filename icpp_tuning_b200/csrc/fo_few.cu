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
  // As many CTAs as are resident at once, two a SM: one CTA keeps 110 KB under way, 43 B/ns of
  // HBM; but K blocks enough that the exchange of the sums stays small beside them.  Measured,
  // for 1, 2, 4, 8 CTAs a tile: gated product 4096 x 16384 (128 tiles), one token 51.6, 45.3,
  // 50.6, 55.8 us, 24 tokens 52.9, 51.1, 57.0, 65.3; 2048 x 8192 (64 tiles) 22.5, 20.3, 17.2,
  // 22.1; block 1 x 1024 x 4096 (32 tiles, 16 K blocks) 16.7, 15.2, 13.8, 14.5; blocks' second
  // product alone changed, 1 x 4096 x 16384 132, 98, 83, 79; dh 64 x 1024 x 4096 42, 34, 21, 17.
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
