// fo_skinny.cu -- instantiations and launch rule of the few-token products, and the C entries
// of the 4-bit weights.
#include "fo_host.cuh"
#include "fo_skinny.cuh"
#include "../../include/b200fo.h"

namespace fo {
namespace {

template <int FMT, bool GATED, int NT, int DT>
cudaError_t launch(const SkinnyParams& p, int sms, cudaStream_t stream) {
  using S = SkinnyShape<FMT, GATED>;
  static std::atomic<uint64_t> opted{0};
  const int tiles = (p.N + S::kFeatures - 1) / S::kFeatures;
  const int chunks = (p.T + 8 * NT - 1) / (8 * NT);
  const int steps = (p.K + S::kStep - 1) / S::kStep;
  // Split K over a cluster until the grid covers the SMs twice, as long as every warp
  // keeps two steps or more.
  int Q = 1;
  while (Q < 8 && static_cast<long long>(tiles) * chunks * Q < 2 * sms && steps >= S::kWarps * Q * 4) Q *= 2;
  const int smem = S::smem_bytes(NT, p.groups, p.zero[0] != nullptr);
  return launch_pdl(fo_skinny_kernel<FMT, GATED, NT, DT>, opted, dim3(tiles * Q, chunks), dim3(256), smem, Q, stream, p);
}

template <int FMT, bool GATED, int DT>
cudaError_t by_tokens(const SkinnyParams& p, int sms, cudaStream_t stream) {
  if (p.T <= 8) return launch<FMT, GATED, 1, DT>(p, sms, stream);
  if (FMT == W_KN || p.T <= 16) return launch<FMT, GATED, 2, DT>(p, sms, stream);
  if constexpr (FMT != W_KN) {
    if (p.T <= 32) return launch<FMT, GATED, 4, DT>(p, sms, stream);
    return launch<FMT, GATED, 8, DT>(p, sms, stream);
  }
  return cudaErrorInvalidValue;
}

template <int DT>
cudaError_t by_format(int fmt, bool gated, const SkinnyParams& p, int sms, cudaStream_t s) {
  if (fmt == W_NK) return gated ? by_tokens<W_NK, true, DT>(p, sms, s) : by_tokens<W_NK, false, DT>(p, sms, s);
  if (fmt == W_KN) return gated ? by_tokens<W_KN, true, DT>(p, sms, s) : by_tokens<W_KN, false, DT>(p, sms, s);
  return gated ? by_tokens<W_Q4, true, DT>(p, sms, s) : by_tokens<W_Q4, false, DT>(p, sms, s);
}

}  // namespace

int gate_act_of(int act) {
  switch (act) {
    case FO_GATE_SILU: return ACT_SILU;
    case FO_GATE_GELU_TANH: return ACT_GELU_TANH;
    case FO_GATE_GELU_ERF: return ACT_GELU_ERF;
    default: return ACT_RELU;
  }
}

cudaError_t launch_skinny(int fmt, bool gated, int dt, const SkinnyParams& p, int sms, cudaStream_t stream) {
  return dt == DT_BF16 ? by_format<DT_BF16>(fmt, gated, p, sms, stream) : by_format<DT_F16>(fmt, gated, p, sms, stream);
}

namespace {

constexpr int kMaxGroups = 1024;  // scales of 32 rows, with zeros, beside the ring in shared memory

int check_weight(const FoW4* w, int64_t N, int64_t K, const char* name) {
  if (w->q == nullptr || w->scales == nullptr || !host_aligned16(w->q))
    return host_fail(FO_EINVAL, "%s: q and scales must be device pointers, q 16-byte aligned", name);
  if (w->group <= 0 || w->group % 32 != 0) return host_fail(FO_EINVAL, "%s: group must be a positive multiple of 32, got %d", name, w->group);
  const int64_t groups = (K + w->group - 1) / w->group;
  if (groups > kMaxGroups)
    return host_fail(FO_EUNSUPPORTED, "%s: %lld groups a row exceed %d", name, static_cast<long long>(groups), kMaxGroups);
  if (w->ldq < K / 2 || w->ldq % 16 != 0)
    return host_fail(FO_EINVAL, "%s: ldq must be a multiple of 16 bytes and >= K / 2, got %lld", name, static_cast<long long>(w->ldq));
  if (w->lds < groups || (w->zeros != nullptr && w->ldz < groups))
    return host_fail(FO_EINVAL, "%s: rows of scales or zeros are shorter than the %lld groups", name, static_cast<long long>(groups));
  (void)N;
  return FO_OK;
}

int check_sizes(int64_t T, int64_t N, int64_t K, int dtype) {
  if (T < 0 || N < 0 || K < 0) return host_fail(FO_EINVAL, "negative problem size");
  if (T > (1ll << 19) || N > (1ll << 27) || K > (1ll << 27)) return host_fail(FO_EINVAL, "problem too large");
  if (dtype != FO_DT_F16 && dtype != FO_DT_BF16) return host_fail(FO_EINVAL, "dtype must be FO_DT_F16 or FO_DT_BF16");
  if (K % 32 != 0) return host_fail(FO_EINVAL, "4-bit rows hold whole 16-byte blocks of 32 weights: K = %lld", static_cast<long long>(K));
  return FO_OK;
}

void set_weight(SkinnyParams* p, int m, const FoW4* w) {
  p->w[m] = w->q, p->ldw[m] = w->ldq;
  p->scale[m] = w->scales, p->lds[m] = w->lds;
  p->zero[m] = static_cast<const unsigned char*>(w->zeros), p->ldz[m] = w->ldz;
}

int check_rows(const void* a, int64_t ld, int64_t cols, const char* name) {
  if (a == nullptr || !host_aligned16(a)) return host_fail(FO_EINVAL, "%s must be a 16-byte aligned device pointer", name);
  if (ld % 8 != 0 || ld < cols) return host_fail(FO_EINVAL, "the row stride of %s must be a multiple of 8 and >= %lld", name, static_cast<long long>(cols));
  return FO_OK;
}

}  // namespace
}  // namespace fo

extern "C" int fo_matvec_w4(const FoMatvecW4Desc* d, void* stream) {
  using namespace fo;
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (int rc = check_sizes(d->T, d->N, d->K, d->dtype)) return rc;
  if (d->act != FO_GATE_NONE && (d->act < FO_GATE_SILU || d->act > FO_GATE_RELU)) return host_fail(FO_EINVAL, "bad activation %d", d->act);
  const bool gated = d->act != FO_GATE_NONE;
  if (d->T == 0 || d->N == 0) return host_ok();
  if (d->K == 0) return host_fail(FO_EINVAL, "K must be positive");
  if (int rc = check_weight(&d->w, d->N, d->K, "w")) return rc;
  if (gated) {
    if (int rc = check_weight(&d->w_up, d->N, d->K, "w_up")) return rc;
    if (d->w.group != d->w_up.group || (d->w.zeros == nullptr) != (d->w_up.zeros == nullptr))
      return host_fail(FO_EINVAL, "both weights of a gated product share the group size and whether they have zeros");
    if (d->bias != nullptr) return host_fail(FO_EINVAL, "a gated product has no bias");
  }
  if (int rc = check_rows(d->x, d->ldx, d->K, "x")) return rc;
  if (d->out == nullptr || d->ldo < d->N) return host_fail(FO_EINVAL, "out must be a device pointer with rows of N values or more");
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  SkinnyParams p = {};
  p.x = d->x, p.ldx = d->ldx, p.T = static_cast<int>(d->T), p.N = static_cast<int>(d->N), p.K = static_cast<int>(d->K);
  set_weight(&p, 0, &d->w);
  if (gated) set_weight(&p, 1, &d->w_up);
  p.group = d->w.group, p.groups = static_cast<int>((d->K + d->w.group - 1) / d->w.group);
  p.scale_vec = p.groups % 8 == 0, p.zero_vec = p.groups % 16 == 0;
  for (int m = 0; m < (gated ? 2 : 1); ++m) {
    p.scale_vec = p.scale_vec && host_aligned16(p.scale[m]) && p.lds[m] % 8 == 0;
    p.zero_vec = p.zero_vec && host_aligned16(p.zero[m]) && p.ldz[m] % 16 == 0;
  }
  p.bias = d->bias, p.out = d->out, p.ldo = d->ldo;
  p.act = gate_act_of(d->act);
  const cudaError_t e = launch_skinny(W_Q4, gated, d->dtype == FO_DT_BF16 ? DT_BF16 : DT_F16, p, hd.sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(1);
  return host_ok();
}
