// fo_ffn.cu -- launches and C entries of the gated feed-forward block.
#include <cstring>

#include "fo_few.cuh"
#include "fo_host.cuh"
#include "../../include/b200fo.h"

namespace fo {
namespace {

template <int EPI, int ACT, int DT>
cudaError_t launch_ffn(const FfnMaps& maps, const FfnParams& p, int pairs, cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0};
  return launch_pdl(fo_ffn_kernel<EPI, ACT, DT>, opted, dim3(2 * (p.units < pairs ? p.units : pairs)), dim3(320), kFfnSmem, 2, stream,
                    maps, p);
}

template <int EPI, int DT>
cudaError_t by_act(int act, const FfnMaps& m, const FfnParams& p, int pairs, cudaStream_t s) {
  switch (act) {
    case FO_GATE_SILU: return launch_ffn<EPI, ACT_SILU, DT>(m, p, pairs, s);
    case FO_GATE_GELU_TANH: return launch_ffn<EPI, ACT_GELU_TANH, DT>(m, p, pairs, s);
    case FO_GATE_GELU_ERF: return launch_ffn<EPI, ACT_GELU_ERF, DT>(m, p, pairs, s);
    default: return launch_ffn<EPI, ACT_RELU, DT>(m, p, pairs, s);
  }
}

cudaError_t launch(int epi, int act, const FfnMaps& m, const FfnParams& p, int pairs, cudaStream_t s) {
  if (epi == FFN_GRADS)
    return p.bf16 ? launch_ffn<FFN_GRADS, ACT_NONE, DT_BF16>(m, p, pairs, s) : launch_ffn<FFN_GRADS, ACT_NONE, DT_F16>(m, p, pairs, s);
  if (epi == FFN_GATED) return p.bf16 ? by_act<FFN_GATED, DT_BF16>(act, m, p, pairs, s) : by_act<FFN_GATED, DT_F16>(act, m, p, pairs, s);
  return p.bf16 ? by_act<FFN_DGATE, DT_BF16>(act, m, p, pairs, s) : by_act<FFN_DGATE, DT_F16>(act, m, p, pairs, s);
}

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t kblocks(int64_t k) { return (k + kBK - 1) / kBK; }

// Parts to cut a product's K into: its tiles of kb K blocks beside `others` K blocks of other
// units on `pairs` CTA pairs.  A cut costs a pass over the parts (about 10 K blocks' time),
// so it has to shorten the longest chain by more.
int cut(int64_t M, int64_t N, int64_t kb, int64_t others, int pairs) {
  const int64_t tiles = (M + kFfnTile - 1) / kFfnTile * ((N + kFfnTile - 1) / kFfnTile);
  int best = 1;
  int64_t best_cost = 0;
  for (int s = 1; s <= kFfnMaxParts && s <= kb; ++s) {
    const int64_t unit = (kb + s - 1) / s + 8, units = tiles * s;
    const int64_t mean = (units * unit + others + pairs - 1) / pairs;
    const int64_t rounds = (units + pairs - 1) / pairs * unit;
    const int64_t cost = (mean > rounds ? mean : rounds) + (s > 1 ? 10 + s : 0);
    if (best_cost == 0 || cost < best_cost) best = s, best_cost = cost;
  }
  return best;
}

// A stored matrix [rows, cols], row-major.
struct Mat {
  const void* p;
  int64_t rows, cols, ld;
};

// One launch being put together: problems in order, then the schedule.
struct Build {
  FfnMaps maps;
  FfnParams p;
  JoinPartsParams join = {};
  int dt;
  int rc = FO_OK;

  explicit Build(int dtype, const HostDevice& hd) : dt(dtype) {
    memset(&maps, 0, sizeof(maps));
    memset(&p, 0, sizeof(p));
    p.bf16 = dtype == FO_DT_BF16;
    p.group_m = 8;
    p.status = hd.status;
    p.timeout_ns = hd.timeout_ns;
  }

  void map(CUtensorMap* m, const Mat& t, uint32_t box_rows, const char* what) {
    if (rc == FO_OK) rc = host_tmap(m, dt, t.p, t.cols, t.rows, static_cast<uint64_t>(t.ld) * 2, 64, box_rows, what);
  }
  // An operand whose rows (kt = false) or columns (kt = true: read transposed) run along the
  // product's M or N.
  void operand(CUtensorMap* m, const Mat& t, bool kt, const char* what) { map(m, t, kt ? 64 : 128, what); }

  FfnProblem& add(int64_t M, int64_t N, int64_t K, int tile_n, int segments) {
    FfnProblem& q = p.prob[p.nprob++];
    q.M = static_cast<int>(M), q.N = static_cast<int>(N);
    q.tiles_m = (q.M + kFfnTile - 1) / kFfnTile;
    q.tiles_n = (q.N + tile_n - 1) / tile_n;
    q.kb0 = static_cast<int>((K + kBK - 1) / kBK);
    q.kb = segments * q.kb0;
    q.parts = 1;
    q.unit0 = p.units;
    p.units += q.tiles_m * q.tiles_n;
    return q;
  }

  // C [M, N] = op(A) op(B) over K (a second pair of operands: a second K segment); parts > 1:
  // fp32 parts in `part`, to be joined into C by join().
  void product(int64_t M, int64_t N, int64_t K, const Mat& a, bool a_t, const Mat& b, bool b_t, const Mat& c,
               const Mat* a1 = nullptr, const Mat* b1 = nullptr, int parts = 1, void* part = nullptr) {
    FfnProblem& q = add(M, N, K, kFfnTile, a1 != nullptr ? 2 : 1);
    const int i = p.nprob - 1;
    q.a_mn = a_t, q.b_mn = b_t;
    operand(&maps.a[i][0], a, a_t, "a product's first operand");
    operand(&maps.b[i][0], b, b_t, "a product's second operand");
    if (a1 != nullptr) {
      operand(&maps.a[i][1], *a1, a_t, "a product's first operand");
      operand(&maps.b[i][1], *b1, b_t, "a product's second operand");
    }
    if (parts > 1) {
      q.parts = parts;
      p.units += (parts - 1) * q.tiles_m * q.tiles_n;
      join = {static_cast<const float*>(part), const_cast<void*>(c.p), q.M, q.N, parts, pad8(N), c.ld};
      if (rc == FO_OK) rc = host_tmap_planes(&maps.c[i], part, N, M, parts, static_cast<uint64_t>(pad8(N)) * 4, "a product's parts");
    } else {
      map(&maps.c[i], c, 32, "a product's output");
    }
  }

  // Launches the products (and the join of the one that was cut).
  cudaError_t run(const HostDevice& hd, cudaStream_t st) {
    cudaError_t e = launch(FFN_GRADS, 0, maps, p, hd.sms / 2, st);
    if (e != cudaSuccess || join.parts < 2) return e;
    static std::atomic<uint64_t> none{0};
    const long long n = static_cast<long long>(join.M) * (join.ldp / 8);
    const long long blocks = (n + 255) / 256, most = 8ll * hd.sms;
    return launch_pdl(p.bf16 ? fo_ffn_join_kernel<DT_BF16> : fo_ffn_join_kernel<DT_F16>, none, dim3(static_cast<unsigned>(blocks < most ? blocks : most)),
                      dim3(256), 0, 1, st, join);
  }

  // Spreads units of different K.  Few: each gets its pair by name, longest first, to the pair
  // with the least work so far (dx of a short batch has few, long tiles; the weight gradients
  // many, short ones).  Many: in turn, but for the pairs that the first problem's longer units
  // leave without one (4096 x 16384 backward, 65 tokens 357 -> 269 us, 512 tokens 445 -> 390;
  // 4096 x 4096 x 8192 1266 -> 1232).
  void schedule(int pairs) {
    if (p.nprob < 2) return;
    if (p.units > kFfnOwners) {
      const FfnProblem &l = p.prob[0], &s = p.prob[1];
      const int long_cost = l.kb / l.parts + 8, short_cost = s.kb / s.parts + 8;
      if (pairs > p.units || long_cost <= short_cost) return;
      p.longs = l.tiles_m * l.tiles_n * l.parts;
      p.over = p.longs % pairs;
      const int rest = pairs - p.over, most = (p.units - p.longs) / rest;
      p.extra = p.over == 0 ? 0 : (long_cost + short_cost / 2) / short_cost;
      if (p.extra > most) p.extra = most;
      return;
    }
    int load[256] = {0};
    if (pairs > 256) pairs = 256;
    if (pairs > p.units) pairs = p.units;
    p.owned = 1;
    for (int i = 0; i < p.nprob; ++i) {
      const FfnProblem& q = p.prob[i];
      for (int t = 0; t < q.tiles_m * q.tiles_n * q.parts; ++t) {
        int best = 0;
        for (int c = 1; c < pairs; ++c)
          if (load[c] < load[best]) best = c;
        p.owner[q.unit0 + t] = static_cast<unsigned char>(best);
        load[best] += q.kb / q.parts + 8;  // the unit's K blocks and about its epilogue
      }
    }
  }
};

int check_mat(const void* p, int64_t ld, int64_t cols, const char* name) {
  if (p == nullptr || !host_aligned16(p)) return host_fail(FO_EINVAL, "%s must be a 16-byte aligned device pointer", name);
  if (ld % 8 != 0 || ld < cols)
    return host_fail(FO_EINVAL, "the row stride of %s must be a multiple of 8 and >= %lld, got %lld", name, static_cast<long long>(cols),
                     static_cast<long long>(ld));
  return FO_OK;
}

int check(const FoGatedFfnDesc* d) {
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (d->T < 0 || d->D < 0 || d->F < 0 || d->N < 0) return host_fail(FO_EINVAL, "negative problem size");
  for (int64_t v : {d->T, d->D, d->F, d->N})
    if (v > (1ll << 27)) return host_fail(FO_EINVAL, "problem too large");
  if (d->dtype != FO_DT_F16 && d->dtype != FO_DT_BF16) return host_fail(FO_EINVAL, "dtype must be FO_DT_F16 or FO_DT_BF16");
  if (d->b_layout != FO_B_KN && d->b_layout != FO_B_NK) return host_fail(FO_EINVAL, "bad b_layout %d", d->b_layout);
  if (d->act < FO_GATE_SILU || d->act > FO_GATE_RELU) return host_fail(FO_EINVAL, "bad activation %d", d->act);
  return FO_OK;
}

int check_weights(const FoGatedFfnDesc* d, bool kn) {
  if (int rc = check_mat(d->x, d->ldx, d->D, "x")) return rc;
  if (int rc = check_mat(d->w_gate, d->ldwg, kn ? d->F : d->D, "w_gate")) return rc;
  if (int rc = check_mat(d->w_up, d->ldwu, kn ? d->F : d->D, "w_up")) return rc;
  return check_mat(d->w_down, d->ldwd, kn ? d->N : d->F, "w_down");
}

int fail_launch(cudaError_t e) { return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e)); }

}  // namespace
}  // namespace fo

namespace fo {
namespace {

// Tokens up to which the short-token kernels run.  Forward at 1024 x 4096, 32 tokens 18.4 us
// there and 24.7 us on CTA pairs (33 tokens; the parts of more would not fit one tile); backward
// 64 tokens 50.1 and 51.2 us, at 4096 x 16384 217 and 269.
constexpr int kFewForward = 32, kFewBackward = 64;

constexpr int kSms = 148;

// How a call runs: on the short-token kernels, or on CTA pairs with the product that has few
// tiles (forward: down, backward: dx) cut into parts.
struct Few {
  bool on;
  FewPlan first, second;  // forward: gated, down; backward: dgate, dx
  int parts;
  size_t matrices, bytes;  // the workspace: h, or dg, du, h; then the parts
};

Few few_of(const FoGatedFfnDesc* d, bool backward) {
  Few f{};
  f.matrices = (static_cast<size_t>(d->T) * pad8(d->F) * 2 * (backward ? 3 : 1) + 255) / 256 * 256;
  f.bytes = f.matrices;
  f.parts = 1;
  f.on = d->T <= (backward ? kFewBackward : kFewForward);
  if (f.on) {
    f.first = backward ? few_plan(FEW_DGATE, d->F, d->T, static_cast<int>(kblocks(d->N)), kSms)
                       : few_plan(FEW_GATED, d->F, d->T, static_cast<int>(kblocks(d->D)), kSms);
    f.second = backward ? few_plan(FEW_PLAIN, d->D, d->T, static_cast<int>(2 * kblocks(d->F)), kSms)
                        : few_plan(FEW_PLAIN, d->N, 2 * d->T, static_cast<int>(kblocks(d->F)), kSms);
    if (!backward) f.matrices *= 2;  // h in two parts
    f.bytes = f.matrices;
    return f;
  }
  if (backward) {
    auto tiles = [](int64_t a, int64_t b) { return (a + kFfnTile - 1) / kFfnTile * ((b + kFfnTile - 1) / kFfnTile); };
    const int64_t others = (2 * tiles(d->D, d->F) + tiles(d->F, d->N)) * (kblocks(d->T) + 8);
    f.parts = cut(d->T, d->D, 2 * kblocks(d->F), others, kSms / 2);
  } else {
    f.parts = cut(d->T, d->N, kblocks(d->F), 0, kSms / 2);
  }
  if (f.parts > 1) f.bytes += static_cast<size_t>(f.parts) * d->T * pad8(backward ? d->D : d->N) * 4;
  return f;
}

struct FewBuild {
  FewMaps m;
  FewParams p;
  int dt, rc = FO_OK;

  FewBuild(const FoGatedFfnDesc* d, const HostDevice& hd, int64_t features, int64_t k, int segments) : dt(d->dtype) {
    memset(&m, 0, sizeof(m));
    memset(&p, 0, sizeof(p));
    p.F = static_cast<int>(features), p.T = static_cast<int>(d->T);
    p.kb0 = static_cast<int>(kblocks(k)), p.kb = segments * p.kb0;
    p.bf16 = d->dtype == FO_DT_BF16;
    p.status = hd.status, p.timeout_ns = hd.timeout_ns;
  }
  void weight(int i, const Mat& w, bool transposed, const char* what) {
    p.a_mn = transposed;
    if (rc == FO_OK) rc = host_tmap(&m.a[i], dt, w.p, w.cols, w.rows, static_cast<uint64_t>(w.ld) * 2, 64, transposed ? 64 : 128, what);
  }
  void token(int i, const Mat& t, int nt, const char* what) {
    if (rc == FO_OK) rc = host_tmap(&m.b[i], dt, t.p, t.cols, t.rows, static_cast<uint64_t>(t.ld) * 2, 64, nt, what);
  }
};

}  // namespace
}  // namespace fo

extern "C" size_t fo_gated_ffn_workspace_size(const FoGatedFfnDesc* d, int32_t backward) {
  if (d == nullptr || d->T <= 0 || d->F <= 0) return 0;
  return fo::few_of(d, backward != 0).bytes;
}

extern "C" int fo_gated_ffn(const FoGatedFfnDesc* d, void* stream) {
  using namespace fo;
  if (int rc = check(d)) return rc;
  if (d->T == 0 || d->N == 0) return host_ok();
  if (d->D == 0 || d->F == 0) return host_fail(FO_EINVAL, "D and F must be positive");
  const bool kn = d->b_layout == FO_B_KN;
  if (int rc = check_weights(d, kn)) return rc;
  if (int rc = check_mat(d->y, d->ldy, d->N, "y")) return rc;
  const bool save = d->g != nullptr;
  if (save != (d->u != nullptr)) return host_fail(FO_EINVAL, "g and u are saved together");
  if (save) {
    if (int rc = check_mat(d->g, d->ldg, d->F, "g")) return rc;
    if (int rc = check_mat(d->u, d->ldu, d->F, "u")) return rc;
  }
  const Few few = few_of(d, false);
  const size_t need = fo_gated_ffn_workspace_size(d, 0);
  if (d->workspace == nullptr || d->workspace_bytes < need || !host_aligned16(d->workspace))
    return host_fail(FO_EINVAL, "the block needs a 16-byte aligned workspace of %zu bytes", need);
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Mat h{d->workspace, d->T, d->F, pad8(d->F)};

  const Mat x{d->x, d->T, d->D, d->ldx};
  const Mat wg{d->w_gate, kn ? d->D : d->F, kn ? d->F : d->D, d->ldwg}, wu{d->w_up, wg.rows, wg.cols, d->ldwu};
  const Mat wd{d->w_down, kn ? d->F : d->N, kn ? d->N : d->F, d->ldwd};
  if (few.on) {
    FewBuild a(d, hd, d->F, d->D, 1), o(d, hd, d->N, d->F, 1);
    a.weight(0, wg, kn, "w_gate"), a.weight(1, wu, kn, "w_up");
    a.token(0, x, few.first.nt, "x");
    const Mat h2{d->workspace, 2 * d->T, d->F, h.ld};
    a.p.out = d->workspace, a.p.ldo = h.ld, a.p.split = 1;
    a.p.g = d->g, a.p.u = d->u, a.p.ldg = d->ldg, a.p.ldu = d->ldu;
    o.weight(0, wd, kn, "w_down");
    o.token(0, h2, few.second.nt, "h");
    o.p.T *= 2, o.p.joint = 1;
    o.p.out = d->y, o.p.ldo = d->ldy;
    o.p.early = 1;
    if (a.rc || o.rc) return a.rc ? a.rc : o.rc;
    cudaError_t e = launch_few(FEW_GATED, d->act, a.m, a.p, few.first, st);
    if (e == cudaSuccess) e = launch_few(FEW_PLAIN, 0, o.m, o.p, few.second, st);
    if (e != cudaSuccess) return fail_launch(e);
    host_count_launches(2);
    return host_ok();
  }

  Build b(d->dtype, hd);
  FfnProblem& q = b.add(d->T, d->F, d->D, kFfnTile / 2, 1);
  q.b_mn = kn;
  b.operand(&b.maps.a[0][0], x, false, "x");
  b.operand(&b.maps.b[0][0], wg, kn, "w_gate");
  b.operand(&b.maps.b[0][1], wu, kn, "w_up");
  b.map(&b.maps.c[0], h, 32, "h");
  b.p.save = save;
  if (save) {
    b.map(&b.maps.c[1], {d->g, d->T, d->F, d->ldg}, 32, "g");
    b.map(&b.maps.c[2], {d->u, d->T, d->F, d->ldu}, 32, "u");
  }
  if (b.rc) return b.rc;
  cudaError_t e = launch(FFN_GATED, d->act, b.maps, b.p, hd.sms / 2, st);
  if (e != cudaSuccess) return fail_launch(e);

  Build y(d->dtype, hd);
  y.product(d->T, d->N, d->F, h, false, wd, kn, {d->y, d->T, d->N, d->ldy}, nullptr, nullptr, few.parts,
            static_cast<char*>(d->workspace) + few.matrices);
  if (y.rc) return y.rc;
  e = y.run(hd, st);
  if (e != cudaSuccess) return fail_launch(e);
  host_count_launches(few.parts > 1 ? 3 : 2);
  return host_ok();
}

extern "C" int fo_gated_ffn_backward(const FoGatedFfnDesc* d, void* stream) {
  using namespace fo;
  if (int rc = check(d)) return rc;
  if (d->D == 0 || d->F == 0 || d->N == 0) return host_fail(FO_EINVAL, "D, F and N must be positive");
  const bool kn = d->b_layout == FO_B_KN;
  if (int rc = check_mat(d->dw_gate, d->lddwg, kn ? d->F : d->D, "dw_gate")) return rc;
  if (int rc = check_mat(d->dw_up, d->lddwu, kn ? d->F : d->D, "dw_up")) return rc;
  if (int rc = check_mat(d->dw_down, d->lddwd, kn ? d->N : d->F, "dw_down")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  HostDevice hd;
  const int64_t up_rows = kn ? d->D : d->F, up_cols = kn ? d->F : d->D;
  const int64_t down_rows = kn ? d->F : d->N, down_cols = kn ? d->N : d->F;
  if (d->T == 0) {  // no tokens: the weight gradients are empty sums
    if (int rc = host_device(&hd)) return rc;
    if (cudaMemset2DAsync(d->dw_gate, d->lddwg * 2, 0, up_cols * 2, up_rows, st) != cudaSuccess ||
        cudaMemset2DAsync(d->dw_up, d->lddwu * 2, 0, up_cols * 2, up_rows, st) != cudaSuccess ||
        cudaMemset2DAsync(d->dw_down, d->lddwd * 2, 0, down_cols * 2, down_rows, st) != cudaSuccess)
      return host_fail(FO_ECUDA, "clearing a weight gradient failed");
    return host_ok();
  }
  if (int rc = check_weights(d, kn)) return rc;
  if (int rc = check_mat(d->dy, d->lddy, d->N, "dy")) return rc;
  if (int rc = check_mat(d->g, d->ldg, d->F, "g")) return rc;
  if (int rc = check_mat(d->u, d->ldu, d->F, "u")) return rc;
  if (int rc = check_mat(d->dx, d->lddx, d->D, "dx")) return rc;
  const Few few = few_of(d, true);
  const size_t need = fo_gated_ffn_workspace_size(d, 1);
  if (d->workspace == nullptr || d->workspace_bytes < need || !host_aligned16(d->workspace))
    return host_fail(FO_EINVAL, "the backward pass needs a 16-byte aligned workspace of %zu bytes", need);
  if (int rc = host_device(&hd)) return rc;
  const int64_t ldf = pad8(d->F);
  char* ws = static_cast<char*>(d->workspace);
  const Mat dg{ws, d->T, d->F, ldf}, du{ws + d->T * ldf * 2, d->T, d->F, ldf}, h{ws + 2 * d->T * ldf * 2, d->T, d->F, ldf};
  const Mat x{d->x, d->T, d->D, d->ldx}, dy{d->dy, d->T, d->N, d->lddy};
  const Mat wg{d->w_gate, up_rows, up_cols, d->ldwg}, wu{d->w_up, up_rows, up_cols, d->ldwu};
  const Mat wd{d->w_down, down_rows, down_cols, d->ldwd};

  cudaError_t e;
  if (few.on) {
    FewBuild a(d, hd, d->F, d->N, 1), o(d, hd, d->D, d->F, 2);
    a.weight(0, wd, !kn, "w_down");
    a.token(0, dy, few.first.nt, "dy");
    a.p.out = const_cast<void*>(dg.p), a.p.g = const_cast<void*>(du.p), a.p.u = const_cast<void*>(h.p);
    a.p.ldo = a.p.ldg = a.p.ldu = ldf;
    a.p.sg = d->g, a.p.su = d->u, a.p.ldsg = d->ldg, a.p.ldsu = d->ldu;
    o.weight(0, wg, !kn, "w_gate"), o.weight(1, wu, !kn, "w_up");
    o.token(0, dg, few.second.nt, "dg"), o.token(1, du, few.second.nt, "du");
    o.p.out = d->dx, o.p.ldo = d->lddx;
    o.p.early = 1;
    if (a.rc || o.rc) return a.rc ? a.rc : o.rc;
    e = launch_few(FEW_DGATE, d->act, a.m, a.p, few.first, st);
    if (e == cudaSuccess) e = launch_few(FEW_PLAIN, 0, o.m, o.p, few.second, st);
    if (e != cudaSuccess) return fail_launch(e);
  } else {
    Build b(d->dtype, hd);
    FfnProblem& q = b.add(d->T, d->F, d->N, kFfnTile, 1);
    q.b_mn = !kn;
    b.operand(&b.maps.a[0][0], dy, false, "dy");
    b.operand(&b.maps.b[0][0], wd, !kn, "w_down");
    b.p.dg = const_cast<void*>(dg.p), b.p.du = const_cast<void*>(du.p), b.p.h = const_cast<void*>(h.p), b.p.ldo = ldf;
    b.p.g = d->g, b.p.u = d->u, b.p.ldg = d->ldg, b.p.ldu = d->ldu;
    if (b.rc) return b.rc;
    e = launch(FFN_DGATE, d->act, b.maps, b.p, hd.sms / 2, st);
    if (e != cudaSuccess) return fail_launch(e);
  }

  Build w(d->dtype, hd);
  auto add_dx = [&] {
    w.product(d->T, d->D, d->F, dg, false, wg, !kn, {d->dx, d->T, d->D, d->lddx}, &du, &wu, few.parts, ws + few.matrices);
  };
  auto add_weights = [&] {
    const Mat owg{d->dw_gate, up_rows, up_cols, d->lddwg}, owu{d->dw_up, up_rows, up_cols, d->lddwu};
    const Mat owd{d->dw_down, down_rows, down_cols, d->lddwd};
    if (kn) {
      w.product(d->D, d->F, d->T, x, true, dg, true, owg);
      w.product(d->D, d->F, d->T, x, true, du, true, owu);
      w.product(d->F, d->N, d->T, h, true, dy, true, owd);
    } else {
      w.product(d->F, d->D, d->T, dg, true, x, true, owg);
      w.product(d->F, d->D, d->T, du, true, x, true, owu);
      w.product(d->N, d->F, d->T, dy, true, h, true, owd);
    }
  };
  if (few.on) {
    add_weights();
  } else if (2 * d->F / few.parts >= d->T) {  // longest units first
    add_dx();
    add_weights();
  } else {
    add_weights();
    add_dx();
  }
  if (w.rc) return w.rc;
  w.schedule(hd.sms / 2);
  e = w.run(hd, st);
  if (e != cudaSuccess) return fail_launch(e);
  host_count_launches(few.on || few.parts > 1 ? 3 : 2);
  return host_ok();
}
