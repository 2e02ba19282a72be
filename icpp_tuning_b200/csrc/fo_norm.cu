// fo_norm.cu -- the norms after and before a block, fused with the block's gate and the
// residual scale, forward and backward.
//
// One row x of the residual stream and one row y of the block's output give
//   n = norm_post(y),  r = a x + gate * n,  z = norm_pre(r)
// (norm: v rho w with rho = rsqrt(mean v^2 + eps), or the LayerNorm form with mean and bias).
// Backward, from dr and dz, with rhat and yhat the normalised rows and means over the row:
//   c = dz w_pre,  t = dr + rho_r (c - [mean c] - rhat mean(c rhat)),  dx = a t,
//   dn = gate t,   e = dn w_post,  dy = rho_y (e - [mean e] - yhat mean(e yhat)),
//   dw_pre = sum dz rhat, dw_post = sum dn yhat, db_* = sum dz, sum dn, dgate = sum t n
// ([.] in the LayerNorm form only; sums over rows).
//
// W warps own a row and hold all of it in registers (thread i the columns
// (v * 32 W + i) * VEC ..), so each input value crosses HBM once and each output once: both
// kernels are bound by HBM.  Statistics are fp32 and two-pass over the registers (mean,
// then centred squares).
#include "fo_host.cuh"
#include "fo_kernel.cuh"
#include "../../include/b200fo.h"

namespace fo {
namespace {

struct NormParams {
  const void *y, *x, *dr, *dz;
  void *r, *z, *dy, *dx;  // r: output forward, input backward
  const void *w_post, *b_post, *w_pre, *b_pre, *gate;
  long long ldy, ldx, ldr, ldz, lddr, lddz, lddy, lddx, ldgate;
  int T, D;
  int rows_per_gate;  // rows sharing one gate row (T for a gate vector)
  int vec_dtype, layer;
  float scale, eps;
  // backward: units of chunk_rows rows inside one gate group; partial sums of worker w in
  // part_w[k][w][ldp] (k: w_pre, w_post, b_pre, b_post), of unit u in part_g[u][ldp]
  int groups, chunks, chunk_rows, workers;
  int ldp;
  float *part_w, *part_g;
};

template <int DT, int VEC>
struct RowVec {  // VEC values of a row as stored (16-bit)
  uint32_t u[VEC == 8 ? 4 : 1];
  __device__ __forceinline__ void load(const void* row, int c, int D) {
    if constexpr (VEC == 8) {
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (c < D) q = __ldg(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(row) + c));
      u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
    } else {
      u[0] = c < D ? __ldg(static_cast<const unsigned short*>(row) + c) : 0u;
    }
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2<DT>(u[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    } else {
      f[0] = unpack2<DT>(u[0]).x;
    }
  }
};

template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void* row, int c, int D, const float (&f)[VEC]) {
  if (c >= D) return;
  unsigned short* p = static_cast<unsigned short*>(row) + c;
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
  } else {
    *p = static_cast<unsigned short>(pack2<DT>(f[0], 0.f) & 0xFFFFu);
  }
}

// VEC values of a parameter vector (`fill` where the vector is absent or c is past D).
template <int VEC>
__device__ __forceinline__ void load_param(const void* ptr, int dt, int c, int D, float fill, float (&f)[VEC]) {
  if (ptr == nullptr || c >= D) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = fill;
  } else if constexpr (VEC == 8) {
    load_vec8(ptr, dt, c, f);
  } else {
    f[0] = load_vec(ptr, dt, c);
  }
}

__device__ __forceinline__ const void* vec_at(const void* ptr, int dt, long long i) {
  return ptr == nullptr ? nullptr : static_cast<const char*>(ptr) + i * (dt == DT_F32 ? 4 : 2);
}

// Sums of N values over the W warps of a row.  Rounds alternate between two halves of the
// scratch: a warp enters round k + 2 only after every warp has read round k (the barrier of
// round k + 1 lies between), so one barrier a round is enough.
template <int W, int N>
struct RowSum {
  float* red;  // [2][N][W] of this row group
  int round, bar;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (W > 1) {
      float* s = red + round * N * W;
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * W + (threadIdx.x >> 5)] = v[i];
      named_bar_sync(bar, 32 * W);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) t += s[i * W + w];
        v[i] = t;
      }
      round ^= 1;
    }
  }
};

constexpr int rows_per_cta(int W) { return W >= 4 ? 1 : 4 / W; }

// hat[] = the normalised values of v[] (v itself on return is v - mean in the LayerNorm
// form); returns rho.  Columns past D hold 0 and stay 0.
template <int VEC, int NV, int W, class Sum>
__device__ __forceinline__ float normalise(float (&v)[NV][VEC], const NormParams& p, Sum& sum, int tid) {
  const float inv = 1.0f / static_cast<float>(p.D);
  if (p.layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[j][i];
    sum(s);
    const float mean = s[0] * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = (j * 32 * W + tid) * VEC < p.D;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = in ? v[j][i] - mean : 0.f;
    }
  }
  float q[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[0] = fmaf(v[j][i], v[j][i], q[0]);
  sum(q);
  return rsqrtf(fmaf(q[0], inv, p.eps));
}

template <int DT, int W, int NV, int VEC>
__global__ void __launch_bounds__(32 * W * rows_per_cta(W)) fo_norm_fwd_kernel(const NormParams p) {
  __shared__ float red[rows_per_cta(W) * 2 * W];
  const int tid = threadIdx.x;
  RowSum<W, 1> sum{red + threadIdx.y * 2 * W, 0, 1 + static_cast<int>(threadIdx.y)};
  griddep_launch_dependents();
  griddep_wait();
  for (int row = blockIdx.x * rows_per_cta(W) + threadIdx.y; row < p.T; row += gridDim.x * rows_per_cta(W)) {
    const unsigned short* yr = static_cast<const unsigned short*>(p.y) + row * p.ldy;
    const unsigned short* xr = static_cast<const unsigned short*>(p.x) + row * p.ldx;
    RowVec<DT, VEC> yv[NV], xv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) yv[j].load(yr, (j * 32 * W + tid) * VEC, p.D);
#pragma unroll
    for (int j = 0; j < NV; ++j) xv[j].load(xr, (j * 32 * W + tid) * VEC, p.D);
    float v[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) yv[j].get(v[j]);
    float rho = 1.f;
    if (p.w_post != nullptr) rho = normalise<VEC, NV, W>(v, p, sum, tid);
    const void* gate = p.gate == nullptr ? nullptr : vec_at(p.gate, p.vec_dtype, row / p.rows_per_gate * p.ldgate);
    unsigned short* rr = static_cast<unsigned short*>(p.r) + row * p.ldr;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * W + tid) * VEC;
      float w[VEC], b[VEC], g[VEC], x[VEC];
      load_param(p.w_post, p.vec_dtype, c, p.D, 1.f, w);
      load_param(p.b_post, p.vec_dtype, c, p.D, 0.f, b);
      load_param(gate, p.vec_dtype, c, p.D, 1.f, g);
      xv[j].get(x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = fmaf(p.scale, x[i], g[i] * fmaf(v[j][i] * rho, w[i], b[i]));
      store_vec<DT, VEC>(rr, c, p.D, v[j]);
    }
    rho = normalise<VEC, NV, W>(v, p, sum, tid);
    unsigned short* zr = static_cast<unsigned short*>(p.z) + row * p.ldz;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 * W + tid) * VEC;
      float w[VEC], b[VEC];
      load_param(p.w_pre, p.vec_dtype, c, p.D, 1.f, w);
      load_param(p.b_pre, p.vec_dtype, c, p.D, 0.f, b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = fmaf(v[j][i] * rho, w[i], b[i]);
      store_vec<DT, VEC>(zr, c, p.D, v[j]);
    }
  }
}

// BIAS: the bias gradients are accumulated too.
template <int DT, int W, int NV, int VEC, bool BIAS>
__global__ void __launch_bounds__(32 * W * rows_per_cta(W)) fo_norm_bwd_kernel(const NormParams p) {
  __shared__ float red[rows_per_cta(W) * 2 * 3 * W];
  const int tid = threadIdx.x;
  RowSum<W, 3> sum3{red + threadIdx.y * 2 * 3 * W, 0, 1 + static_cast<int>(threadIdx.y)};
  const int worker = blockIdx.x * rows_per_cta(W) + threadIdx.y;
  const float inv = 1.0f / static_cast<float>(p.D);
  float a_wpre[NV][VEC] = {}, a_wpost[NV][VEC] = {}, a_gate[NV][VEC] = {};
  float a_bpre[BIAS ? NV : 1][VEC] = {}, a_bpost[BIAS ? NV : 1][VEC] = {};
  griddep_launch_dependents();
  griddep_wait();
  for (int u = worker; u < p.groups * p.chunks; u += p.workers) {
    const int grp = u / p.chunks, chunk = u - grp * p.chunks;
    const int lo = grp * p.rows_per_gate + chunk * p.chunk_rows;
    const int hi = min((grp + 1) * p.rows_per_gate, lo + p.chunk_rows);
    const void* gate = p.gate == nullptr ? nullptr : vec_at(p.gate, p.vec_dtype, grp * p.ldgate);
    for (int row = lo; row < hi; ++row) {
      const unsigned short* rp[4] = {static_cast<const unsigned short*>(p.r) + row * p.ldr,
                                     static_cast<const unsigned short*>(p.dz) + row * p.lddz,
                                     static_cast<const unsigned short*>(p.y) + row * p.ldy,
                                     static_cast<const unsigned short*>(p.dr) + row * p.lddr};
      RowVec<DT, VEC> in[4][NV];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < NV; ++j) in[k][j].load(rp[k], (j * 32 * W + tid) * VEC, k == 3 && p.dr == nullptr ? 0 : p.D);
      float mean_r = 0.f, mean_y = 0.f, mean_c = 0.f;
      if (p.layer) {
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float r[VEC], z[VEC], y[VEC], w[VEC];
          in[0][j].get(r), in[1][j].get(z), in[2][j].get(y);
          load_param(p.w_pre, p.vec_dtype, (j * 32 * W + tid) * VEC, p.D, 1.f, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[0] += r[i], s[1] += y[i], s[2] = fmaf(z[i], w[i], s[2]);
        }
        sum3(s);
        mean_r = s[0] * inv, mean_y = p.w_post != nullptr ? s[1] * inv : 0.f, mean_c = s[2] * inv;
      }
      float q[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float r[VEC], z[VEC], y[VEC], w[VEC];
        in[0][j].get(r), in[1][j].get(z), in[2][j].get(y);
        const int c = (j * 32 * W + tid) * VEC;
        load_param(p.w_pre, p.vec_dtype, c, p.D, 1.f, w);
        if (c < p.D)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float rc = r[i] - mean_r, yc = y[i] - mean_y;
            q[0] = fmaf(rc, rc, q[0]);
            q[1] = fmaf(yc, yc, q[1]);
            q[2] = fmaf(z[i] * w[i], rc, q[2]);
          }
      }
      sum3(q);
      const float rho_r = rsqrtf(fmaf(q[0], inv, p.eps));
      const float rho_y = p.w_post != nullptr ? rsqrtf(fmaf(q[1], inv, p.eps)) : 1.f;
      const float m_c = q[2] * inv * rho_r;  // mean(c rhat)
      float t[NV][VEC];
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * 32 * W + tid) * VEC;
        float r[VEC], z[VEC], y[VEC], d[VEC], w[VEC], wp[VEC], bp[VEC], g[VEC], dx[VEC];
        in[0][j].get(r), in[1][j].get(z), in[2][j].get(y), in[3][j].get(d);
        load_param(p.w_pre, p.vec_dtype, c, p.D, 1.f, w);
        load_param(p.w_post, p.vec_dtype, c, p.D, 1.f, wp);
        load_param(p.b_post, p.vec_dtype, c, p.D, 0.f, bp);
        load_param(gate, p.vec_dtype, c, p.D, 1.f, g);
        const bool inb = c < p.D;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float rh = inb ? (r[i] - mean_r) * rho_r : 0.f;
          const float yh = inb ? (y[i] - mean_y) * rho_y : 0.f;
          const float tt = inb ? d[i] + rho_r * (fmaf(z[i], w[i], -mean_c) - rh * m_c) : 0.f;
          dx[i] = p.scale * tt;
          a_wpre[j][i] = fmaf(z[i], rh, a_wpre[j][i]);
          const float dn = g[i] * tt;
          a_wpost[j][i] = fmaf(dn, yh, a_wpost[j][i]);
          a_gate[j][i] = fmaf(tt, fmaf(yh, wp[i], bp[i]), a_gate[j][i]);
          if constexpr (BIAS) {
            a_bpre[j][i] += z[i];
            a_bpost[j][i] += dn;
          }
          t[j][i] = dn * wp[i];  // e
          s[0] = fmaf(t[j][i], yh, s[0]);
          s[1] += t[j][i];
        }
        store_vec<DT, VEC>(static_cast<unsigned short*>(p.dx) + row * p.lddx, c, p.D, dx);
      }
      float m_e = 0.f, mean_e = 0.f;
      if (p.w_post != nullptr) {
        sum3(s);
        m_e = s[0] * inv;
        mean_e = p.layer ? s[1] * inv : 0.f;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float y[VEC];
        in[2][j].get(y);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (p.w_post != nullptr) t[j][i] = rho_y * (t[j][i] - mean_e - (y[i] - mean_y) * rho_y * m_e);
        store_vec<DT, VEC>(static_cast<unsigned short*>(p.dy) + row * p.lddy, (j * 32 * W + tid) * VEC, p.D, t[j]);
      }
    }
    if (p.gate != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = (j * 32 * W + tid) * VEC + i;
          if (c < p.D) p.part_g[static_cast<long long>(u) * p.ldp + c] = a_gate[j][i];
          a_gate[j][i] = 0.f;
        }
    }
  }
  if (worker < p.workers) {
    const long long stride = static_cast<long long>(p.workers) * p.ldp;
    float* base = p.part_w + static_cast<long long>(worker) * p.ldp;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (j * 32 * W + tid) * VEC + i;
        if (c >= p.D) continue;
        base[c] = a_wpre[j][i];
        if (p.w_post != nullptr) base[stride + c] = a_wpost[j][i];
        if constexpr (BIAS) {
          base[2 * stride + c] = a_bpre[j][i];
          base[3 * stride + c] = a_bpost[j][i];
        }
      }
  }
}

// Joins the partial sums in a fixed order: block (output row, 64 columns).  Output rows
// 0..3 are the parameter vectors (all workers), 4 + g the gate rows (their own chunks).
struct JoinParams {
  const float *part_w, *part_g;
  void* out[5];  // dw_pre, dw_post, db_pre, db_post, dgate; null: not wanted
  int workers, chunks, ldp, D, vec_dtype;
};

constexpr int kJoinSplit = 16;

__global__ void __launch_bounds__(16 * kJoinSplit) fo_norm_join_kernel(const JoinParams p) {
  __shared__ float4 red[kJoinSplit][16];
  griddep_launch_dependents();
  griddep_wait();
  const int k = min(static_cast<int>(blockIdx.x), 4);
  if (p.out[k] == nullptr) return;
  const int g = static_cast<int>(blockIdx.x) - 4;
  const int n = k < 4 ? p.workers : p.chunks;
  const float* src = k < 4 ? p.part_w + static_cast<long long>(k) * p.workers * p.ldp
                           : p.part_g + static_cast<long long>(g) * p.chunks * p.ldp;
  const int lane = threadIdx.x & 15, split = threadIdx.x >> 4;
  const int c = blockIdx.y * 64 + lane * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < p.ldp) {
#pragma unroll 4
    for (int i = split; i < n; i += kJoinSplit) {
      const float4 q = __ldcg(reinterpret_cast<const float4*>(src + static_cast<long long>(i) * p.ldp + c));
      a.x += q.x, a.y += q.y, a.z += q.z, a.w += q.w;
    }
  }
  red[split][lane] = a;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int cc = blockIdx.y * 64 + threadIdx.x;
    float t = 0.f;
#pragma unroll
    for (int s = 0; s < kJoinSplit; ++s) t += reinterpret_cast<const float*>(red[s])[threadIdx.x];
    if (cc < p.D) {
      const long long at = (k < 4 ? 0 : static_cast<long long>(g) * p.D) + cc;
      if (p.vec_dtype == DT_F32) static_cast<float*>(p.out[k])[at] = t;
      if (p.vec_dtype == DT_BF16) static_cast<__nv_bfloat16*>(p.out[k])[at] = __float2bfloat16_rn(t);
      if (p.vec_dtype == DT_F16) static_cast<__half*>(p.out[k])[at] = __float2half_rn(t);
    }
  }
}

// ---------------------------------------------------------------------- host
using NormKernel = void (*)(const NormParams);

struct Shape {
  NormKernel kern;
  int warps;
  std::atomic<int>* per_sm;  // resident CTAs of a SM, queried once
};

template <int DT, int W, int NV, int VEC>
Shape fwd_entry() {
  static std::atomic<int> n{0};
  return {fo_norm_fwd_kernel<DT, W, NV, VEC>, W, &n};
}

template <int DT, int W, int NV, int VEC, bool BIAS>
Shape bwd_entry() {
  return {fo_norm_bwd_kernel<DT, W, NV, VEC, BIAS>, W, nullptr};
}

// The row layout for D columns: the fewest warps whose threads hold at most NV vectors of
// 8 (32 columns a thread forward, 16 backward, where each column also carries its sums).
template <int DT, int VEC>
Shape fwd_shape(int D) {
  constexpr int M = VEC == 8 ? 1 : 8;
  if (D <= 256) return fwd_entry<DT, 1, 1 * M, VEC>();
  if (D <= 512) return fwd_entry<DT, 1, 2 * M, VEC>();
  if (D <= 1024) return fwd_entry<DT, 2, 2 * M, VEC>();
  if (D <= 2048) return fwd_entry<DT, 4, 2 * M, VEC>();
  if (D <= 4096) return fwd_entry<DT, 8, 2 * M, VEC>();
  if (D <= 8192) return fwd_entry<DT, 16, 2 * M, VEC>();
  return fwd_entry<DT, 16, 4 * M, VEC>();
}

template <int DT, int VEC, bool BIAS>
Shape bwd_shape(int D) {
  constexpr int M = VEC == 8 ? 1 : 8;
  if (D <= 256) return bwd_entry<DT, 1, 1 * M, VEC, BIAS>();
  if (D <= 512) return bwd_entry<DT, 1, 2 * M, VEC, BIAS>();
  if (D <= 1024) return bwd_entry<DT, 2, 2 * M, VEC, BIAS>();
  if (D <= 2048) return bwd_entry<DT, 4, 2 * M, VEC, BIAS>();
  if (D <= 4096) return bwd_entry<DT, 8, 2 * M, VEC, BIAS>();
  return bwd_entry<DT, 16, 2 * M, VEC, BIAS>();
}

constexpr int kMaxFwd = 16384, kMaxBwd = 8192;

int esize(int dt) { return dt == FO_DT_F32 ? 4 : 2; }

// 16-byte loads of every row and vector: the widths, strides and addresses allow them.
bool vectors(const FoBlockNormDesc* d, bool bwd) {
  bool ok = d->D % 8 == 0;
  const void* rows[] = {d->y, d->r, bwd ? d->dr : d->x, bwd ? d->dz : d->z, bwd ? d->dy : nullptr, bwd ? d->dx : nullptr};
  const int64_t lds[] = {d->ldy, d->ldr, bwd ? d->lddr : d->ldx, bwd ? d->lddz : d->ldz, bwd ? d->lddy : 0, bwd ? d->lddx : 0};
  for (int i = 0; i < 6; ++i) ok = ok && host_aligned16(rows[i]) && (rows[i] == nullptr || lds[i] % 8 == 0);
  for (const void* v : {d->w_post, d->b_post, d->w_pre, d->b_pre, d->gate}) ok = ok && host_aligned16(v);
  return ok && (d->gate_rows <= 1 || (d->ldgate * esize(d->vec_dtype)) % 16 == 0);
}

int check(const FoBlockNormDesc* d, bool bwd) {
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (d->T < 0 || d->D < 0) return host_fail(FO_EINVAL, "negative problem size");
  if (d->T > (1ll << 31) - 1) return host_fail(FO_EINVAL, "T = %lld exceeds 2^31 - 1", static_cast<long long>(d->T));
  if (d->dtype != FO_DT_F16 && d->dtype != FO_DT_BF16) return host_fail(FO_EINVAL, "dtype must be FO_DT_F16 or FO_DT_BF16");
  if (d->vec_dtype < FO_DT_F16 || d->vec_dtype > FO_DT_F32) return host_fail(FO_EINVAL, "bad vec_dtype %d", d->vec_dtype);
  if (d->norm != FO_NORM_RMS && d->norm != FO_NORM_LAYER) return host_fail(FO_EINVAL, "norm must be FO_NORM_RMS or FO_NORM_LAYER");
  if (!(d->eps >= 0.f)) return host_fail(FO_EINVAL, "eps must be >= 0");
  if (d->w_post == nullptr && d->b_post != nullptr) return host_fail(FO_EINVAL, "b_post without w_post");
  if (d->norm == FO_NORM_RMS && (d->b_post != nullptr || d->b_pre != nullptr))
    return host_fail(FO_EINVAL, "the rms norm has no bias");
  if (d->gate_rows < 0 || (d->gate_rows == 0) != (d->gate == nullptr))
    return host_fail(FO_EINVAL, "gate_rows must be 0 without a gate and >= 1 with one");
  if (d->gate_rows > 0 && d->T % d->gate_rows != 0)
    return host_fail(FO_EINVAL, "gate_rows %lld does not divide T = %lld", static_cast<long long>(d->gate_rows),
                     static_cast<long long>(d->T));
  const int most = bwd ? kMaxBwd : kMaxFwd;
  if (d->D > most) return host_fail(FO_EUNSUPPORTED, "D = %lld exceeds %d", static_cast<long long>(d->D), most);
  return FO_OK;
}

void fill(NormParams* p, const FoBlockNormDesc* d) {
  *p = {};
  p->y = d->y, p->x = d->x, p->dr = d->dr, p->dz = d->dz;
  p->r = d->r, p->z = d->z, p->dy = d->dy, p->dx = d->dx;
  p->w_post = d->w_post, p->b_post = d->b_post, p->w_pre = d->w_pre, p->b_pre = d->b_pre, p->gate = d->gate;
  p->ldy = d->ldy, p->ldx = d->ldx, p->ldr = d->ldr, p->ldz = d->ldz;
  p->lddr = d->lddr, p->lddz = d->lddz, p->lddy = d->lddy, p->lddx = d->lddx, p->ldgate = d->ldgate;
  p->T = static_cast<int>(d->T), p->D = static_cast<int>(d->D);
  p->rows_per_gate = d->gate_rows > 0 ? p->T / static_cast<int>(d->gate_rows) : p->T;
  p->vec_dtype = d->vec_dtype, p->layer = d->norm == FO_NORM_LAYER;
  p->scale = d->residual_scale, p->eps = d->eps;
}

// CTAs of one wave a kernel is launched with (the rows are walked with that stride).
int resident(const Shape& k, int threads, int sms) {
  int n = k.per_sm->load(std::memory_order_relaxed);
  if (n == 0) {
    RelaxedCapture relaxed;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k.kern, threads, 0) != cudaSuccess || n < 1) n = 1;
    k.per_sm->store(n, std::memory_order_relaxed);
  }
  return sms * n;
}

std::atomic<uint64_t> g_no_opt{0};  // these kernels use no dynamic shared memory

// Work split of the backward kernel: one wave of workers, each walking chunks of rows that
// share a gate row.  It goes by 148 SMs whatever the device, so that the workspace's size
// needs no device.

int bwd_warps(int64_t D) {
  return D <= 512 ? 1 : D <= 1024 ? 2 : D <= 2048 ? 4 : D <= 4096 ? 8 : 16;
}

struct BwdPlan {
  int workers, groups, chunks, chunk_rows, ldp;
  size_t bytes;
};

BwdPlan bwd_plan(const FoBlockNormDesc* d) {
  BwdPlan b{};
  const int W = bwd_warps(d->D);
  // 16 warps a SM carry rows at once (one row a CTA of 8 warps: two CTAs)
  const int cap = 148 * (W >= 16 ? 1 : 16 / W);
  b.groups = d->gate_rows > 0 ? static_cast<int>(d->gate_rows) : 1;
  const int rpg = static_cast<int>(d->T / b.groups);
  int chunks = b.groups >= cap ? 1 : cap / b.groups;
  if (chunks > rpg) chunks = rpg;
  if (chunks < 1) chunks = 1;
  b.chunk_rows = (rpg + chunks - 1) / chunks;
  b.chunks = b.chunk_rows > 0 ? (rpg + b.chunk_rows - 1) / b.chunk_rows : 1;
  const long long units = static_cast<long long>(b.groups) * b.chunks;
  b.workers = static_cast<int>(units < cap ? units : cap);
  b.ldp = (static_cast<int>(d->D) + 3) / 4 * 4;
  b.bytes = (4 * static_cast<size_t>(b.workers) + (d->gate_rows > 0 ? static_cast<size_t>(units) : 0)) * b.ldp * sizeof(float);
  return b;
}

}  // namespace
}  // namespace fo

extern "C" int fo_block_norm(const FoBlockNormDesc* d, void* stream) {
  using namespace fo;
  if (int rc = check(d, false)) return rc;
  if (d->T == 0 || d->D == 0) return host_ok();
  if (d->y == nullptr || d->x == nullptr || d->r == nullptr || d->z == nullptr || d->w_pre == nullptr)
    return host_fail(FO_EINVAL, "y, x, w_pre, r and z must be device pointers");
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  NormParams p;
  fill(&p, d);
  const bool v8 = vectors(d, false), bf = d->dtype == FO_DT_BF16;
  const int D = p.D;
  const Shape s = bf ? (v8 ? fwd_shape<DT_BF16, 8>(D) : fwd_shape<DT_BF16, 1>(D))
                     : (v8 ? fwd_shape<DT_F16, 8>(D) : fwd_shape<DT_F16, 1>(D));
  const int R = rows_per_cta(s.warps);
  const long long want = (d->T + R - 1) / R;
  const int most = resident(s, 32 * s.warps * R, hd.sms);
  const cudaError_t e = launch_pdl(s.kern, g_no_opt, dim3(static_cast<unsigned>(want < most ? want : most)),
                                   dim3(32 * s.warps, R), 0, 1, static_cast<cudaStream_t>(stream), p);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(1);
  return host_ok();
}

extern "C" size_t fo_block_norm_backward_workspace_size(const FoBlockNormDesc* d) {
  if (d == nullptr || d->T <= 0 || d->D <= 0 || d->gate_rows < 0) return 0;
  return fo::bwd_plan(d).bytes;
}

extern "C" int fo_block_norm_backward(const FoBlockNormDesc* d, void* stream) {
  using namespace fo;
  if (int rc = check(d, true)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->D == 0) return host_ok();
  const size_t vb = static_cast<size_t>(d->D) * esize(d->vec_dtype);
  if (d->T == 0) {  // no rows: the parameter gradients are empty sums
    HostDevice hd;
    if (int rc = host_device(&hd)) return rc;
    for (void* v : {d->dw_post, d->db_post, d->dw_pre, d->db_pre, d->gate_rows > 0 ? d->dgate : nullptr})
      if (v != nullptr && cudaMemsetAsync(v, 0, v == d->dgate ? vb * d->gate_rows : vb, st) != cudaSuccess)
        return host_fail(FO_ECUDA, "clearing a gradient failed");
    return host_ok();
  }
  if (d->y == nullptr || d->r == nullptr || d->dz == nullptr || d->w_pre == nullptr || d->dy == nullptr || d->dx == nullptr ||
      d->dw_pre == nullptr)
    return host_fail(FO_EINVAL, "y, r, dz, w_pre, dy, dx and dw_pre must be device pointers");
  if ((d->w_post != nullptr && d->dw_post == nullptr) || (d->gate != nullptr && d->dgate == nullptr))
    return host_fail(FO_EINVAL, "w_post needs dw_post, a gate needs dgate");
  const BwdPlan b = bwd_plan(d);
  if (d->workspace == nullptr || d->workspace_bytes < b.bytes || !host_aligned16(d->workspace))
    return host_fail(FO_EINVAL, "the backward pass needs a 16-byte aligned workspace of %zu bytes", b.bytes);
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  NormParams p;
  fill(&p, d);
  p.groups = b.groups, p.chunks = b.chunks, p.chunk_rows = b.chunk_rows, p.workers = b.workers, p.ldp = b.ldp;
  p.part_w = static_cast<float*>(d->workspace);
  p.part_g = p.part_w + 4 * static_cast<size_t>(b.workers) * b.ldp;
  const bool v8 = vectors(d, true), bf = d->dtype == FO_DT_BF16, bias = d->db_post != nullptr || d->db_pre != nullptr;
  const int D = p.D;
  const Shape s = bf ? (v8 ? (bias ? bwd_shape<DT_BF16, 8, true>(D) : bwd_shape<DT_BF16, 8, false>(D))
                           : (bias ? bwd_shape<DT_BF16, 1, true>(D) : bwd_shape<DT_BF16, 1, false>(D)))
                     : (v8 ? (bias ? bwd_shape<DT_F16, 8, true>(D) : bwd_shape<DT_F16, 8, false>(D))
                           : (bias ? bwd_shape<DT_F16, 1, true>(D) : bwd_shape<DT_F16, 1, false>(D)));
  const int R = rows_per_cta(s.warps);
  cudaError_t e = launch_pdl(s.kern, g_no_opt, dim3((b.workers + R - 1) / R), dim3(32 * s.warps, R), 0, 1, st, p);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  JoinParams j{};
  j.part_w = p.part_w, j.part_g = p.part_g;
  j.out[0] = d->dw_pre, j.out[1] = d->w_post != nullptr ? d->dw_post : nullptr, j.out[2] = d->db_pre, j.out[3] = d->db_post;
  j.out[4] = d->gate != nullptr ? d->dgate : nullptr;
  j.workers = b.workers, j.chunks = b.chunks, j.ldp = b.ldp, j.D = D, j.vec_dtype = d->vec_dtype;
  const unsigned outs = 4u + (d->gate != nullptr ? static_cast<unsigned>(b.groups) : 0u);
  e = launch_pdl(fo_norm_join_kernel, g_no_opt, dim3(outs, (D + 63) / 64), dim3(16 * kJoinSplit), 0, 1, st, j);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(2);
  return host_ok();
}
