// fo_w4.cu -- products of a few tokens with 4-bit weights, out[t, n] = sum_k x[t, k] w[n, k],
// w = scale (q - zero) by groups along k: plain (optional bias) or gated, act(x Wg^T) * (x Wu^T).
//
// Bound by the weights' bytes, and close behind by issue: a SM has to open about 46 weights
// a cycle to keep up with HBM.  So
//   * a warp streams 32 rows (16 and their 16 partners of a gated pair) and its tokens' x in
//     steps of 128 k, by 16-byte cp.async into a ring it keeps for itself, and asks for a step's scales one
//     step ahead: no block-wide barrier in the loop, and no load whose latency the loop sees;
//   * one ldmatrix hands every lane the 32-bit words (8 weights each) of a 32-k group: of
//     weight row lane / 4, word lane % 4 -- the fragment layout of mma.m16n8k16 when the k
//     order inside a group is that of the words.  The order is free as long as both operands
//     share it: a word's nibbles pair as (0,4), (1,5), (2,6), (3,7), x to match;
//   * a pair is opened by a shift and one logic operation: in fp16 the bits of q alone are
//     the subnormal q 2^-24, exact, and the scale takes 2^24 back; in bf16 the bits of 128 + q
//     (its subnormals would leave fp32's range).  What stays of an offset, and the zero, leave
//     by a product with sum(x) of the group, which one more MMA with a row of ones gives;
//   * 16 weight rows x 8 tokens an MMA: up to 8 tokens cost what one costs.
// W of a CTA's 8 warps share a tile of rows and split its K (and, for few tiles, the CTAs of
// a cluster): as many as make about 2000 warps, so that each still walks many steps.  Partial
// sums meet in shared memory (distributed across the cluster) and are added in a fixed order.
#include "fo_host.cuh"
#include "fo_math.cuh"
#include "../../include/b200fo.h"

namespace fo {
namespace {

struct W4Params {
  const void* x;
  long long ldx;
  int T, N, K;
  const void* q[2];  // [1]: the up weights of a gated product
  const void* scale[2];
  const unsigned char* zero[2];  // null: 8
  long long ldq[2], lds[2], ldz[2];
  int per32;      // 32-k blocks a group
  uint32_t rcp;   // 2^32 / (steps a group), rounded up: GS 4, groups longer than a step
  int vec;        // four scales (zeros) of a row are read at once
  int share;      // W: warps that share a tile
  const void* bias;
  int act;
  void* out;
  long long ldo;
  // The product between the gated block's two kernels travels as two 16-bit parts, high and
  // low, in rows 2 t and 2 t + 1: written so (split), or read so and added (joint; T rows of
  // x, T / 2 of out).
  int split, joint;
};

template <int DT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float* c) {
  if constexpr (DT == DT_BF16) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  } else {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
}

// Four 8 x 16-byte blocks: lane l gives the address of row l % 8 of block l / 8 and
// gets word l % 4 of row l / 4 of each block.
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&w)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

constexpr int kWarps = 8;

constexpr int kRows = 32;                  // weight rows of a tile: two 16-row MMA blocks
constexpr int kStepW = kRows * 64;         // their bytes in a step
constexpr int kTable = kRows * 40;         // a step's (scale, -scale * offset) pairs, up to 4 a row

// NT: 8-token MMA blocks; XT: tokens the ring has room for.
template <int NT, int XT>
struct W4Shape {
  static constexpr int kStep = kStepW + 256 * XT;
  // three CTAs a SM for a token or two, two up to 16 tokens, else one
  static constexpr int kCtas = XT == 2 ? 3 : NT <= 2 ? 2 : 1;
  static constexpr int kBudget = (XT == 2 ? 73 : NT <= 2 ? 110 : 200) * 1024 / kWarps - kTable;
  static constexpr int kStages = kBudget / kStep < 6 ? kBudget / kStep : 6;
  static constexpr int kRed = kRows * 8 * NT * 4;  // one warp's sums: its idle ring at the end
  static constexpr int kWarp = ((kStages * kStep > kRed ? kStages * kStep : kRed) + kTable + 127) / 128 * 128;  // bytes of a warp
  static constexpr int kSmem = kWarps * kWarp + kRed;
  static_assert(kStages >= 2, "a ring");
};

// GS: 32-k blocks whose sums share a scale in one step (1, 2 or 4; 1 serves any group size).
template <bool GATED, int NT, int XT, int GS, int DT>
__global__ void __launch_bounds__(256, (W4Shape<NT, XT>::kCtas)) fo_w4_kernel(const __grid_constant__ W4Params p) {
  using S = W4Shape<NT, XT>;
  constexpr int ENT = 4 / GS, kOut = GATED ? 16 : 32;         // outputs of a tile
  constexpr float kLeft = DT == DT_BF16 ? 128.f : 0.f;        // offset that stays in the opened weights
  constexpr float kBack = DT == DT_BF16 ? 1.f : 16777216.f;   // what their scale lacks
  constexpr uint32_t kMagic = DT == DT_BF16 ? 0x43004300u : 0u;
  constexpr uint32_t kOne = DT == DT_BF16 ? 0x3F803F80u : 0x3C003C00u;
  extern __shared__ __align__(128) uint8_t smem_w4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  int rank, Q;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(Q));
  const int W = p.share, per_cta = kWarps / W;
  const int tile0 = static_cast<int>(blockIdx.x / Q) * per_cta;
  const int n0 = (tile0 + warp / W) * kOut;
  const int tok0 = static_cast<int>(blockIdx.y) * 8 * NT;
  const int toks = min(8 * NT, p.T - tok0);
  const int steps = (p.K + 127) / 128;
  const int first = rank * W + warp % W, stride = Q * W;  // this warp's steps
  const int mine = n0 < p.N && first < steps ? (steps - first + stride - 1) / stride : 0;
  uint8_t* const own = smem_w4 + warp * S::kWarp;
  const uint32_t ring = smem_u32(own);
  uint8_t* const table = own + S::kWarp - kTable;

  // Sources of this lane.  Rows past N repeat the last one: nothing of them is stored.  Row
  // block b: the gate's and the up weights' 16 rows, or rows 16 b of the one matrix.
  const char* src[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int m = GATED ? c >> 1 : 0, n = n0 + r + 8 * (GATED ? c & 1 : c);
    src[c] = static_cast<const char*>(p.q[m]) + min(n, p.N - 1) * p.ldq[m] + t * 16;
  }
  const unsigned short* xs = static_cast<const unsigned short*>(p.x) + (tok0 + (lane >> 4)) * p.ldx + (lane & 15) * 8;
  // The four 16-byte blocks of a weight row are stored rotated, odd tokens' halves swapped, so
  // that the reads below fall into distinct banks.
  const uint32_t w_at = (r * 4 + (t ^ ((r >> 1) & 3))) * 16;
  const uint32_t x_at = kStepW + ((lane >> 4) * 16 + ((lane & 15) ^ ((lane >> 4) << 2))) * 16;
  int todo = 0;               // steps asked for
  uint32_t put = ring;        // where the next one goes
  auto issue = [&]() {        // this warp's next step (an empty group past the end)
    if (todo < mine) {
      const int s = first + todo * stride;
      // past K: zeros, and nothing is read
      const uint32_t wn = s * 128 + t * 32 < p.K ? 16u : 0u, xn = s * 128 + (lane & 15) * 8 < p.K ? 16u : 0u;
      const int wo = wn ? s * 64 : 0, xo = xn ? s * 128 : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) cp_async_16(put + w_at + c * 512, src[c] + wo, wn);
#pragma unroll
      for (int c = 0; c < XT / 2; ++c) {  // two tokens a copy, 16 blocks each
        if (c > 0 && 2 * c >= toks) break;
        if (2 * c + (lane >> 4) < toks) cp_async_16(put + x_at + c * 512, xs + 2 * c * p.ldx + xo, xn);
      }
    }
    cp_async_commit();
    ++todo;
    put += S::kStep;
    if (put == ring + S::kStages * S::kStep) put = ring;
  };
  // A step's scales and zeros: lane l those of row l.
  const int tm = GATED ? lane >> 4 : 0, tn = min(n0 + (GATED ? lane & 15 : lane), p.N - 1);
  const unsigned short* sc = static_cast<const unsigned short*>(p.scale[tm]) + tn * p.lds[tm];
  const unsigned char* zc = p.zero[tm] == nullptr ? nullptr : p.zero[tm] + tn * p.ldz[tm];
  const int groups = (p.K + p.per32 * 32 - 1) / (p.per32 * 32);
  unsigned short sraw[ENT];
  uint32_t zraw = 0x08080808u;
  auto ask = [&](int s) {
    if (GS == 1 && p.vec && s * 4 + 4 <= groups) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(sc + s * 4));
      sraw[0] = static_cast<unsigned short>(v.x), sraw[1 % ENT] = static_cast<unsigned short>(v.x >> 16);
      sraw[2 % ENT] = static_cast<unsigned short>(v.y), sraw[3 % ENT] = static_cast<unsigned short>(v.y >> 16);
      if (zc != nullptr) zraw = __ldg(reinterpret_cast<const uint32_t*>(zc + s * 4));
      return;
    }
    uint32_t z = 0;
#pragma unroll
    for (int e = 0; e < ENT; ++e) {
      const int at = GS == 4 ? (p.rcp != 0 ? static_cast<int>(__umulhi(static_cast<uint32_t>(s), p.rcp)) : s)
                     : GS == 2 ? s * 2 + e : (s * 4 + e) / p.per32;
      const int g = min(at, groups - 1);  // past K: unused
      sraw[e] = __ldg(sc + g);
      z |= (zc != nullptr ? static_cast<uint32_t>(__ldg(zc + g)) : 8u) << (8 * e);
    }
    zraw = z;
  };

  griddep_wait();
  griddep_launch_dependents();
  if (mine > 0) ask(first);
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue();

  float acc[2][NT][4] = {};
  const float none[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
  // ldmatrix: lane l addresses row l % 8 of row block l / 8
  const uint32_t my_row = (lane >> 3) * 512u + (lane & 7) * 64u, my_rot = ((lane & 7) >> 1) & 3;
  const uint32_t my_x = kStepW + r * 256u, x_rot = (r & 1) << 2;
  uint32_t stage = ring;
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();  // other lanes' copies, and their reads of the slot and the table refilled next
#pragma unroll
    for (int e = 0; e < ENT; ++e) {
      const float v = unpack2<DT>(sraw[e]).x, z = static_cast<float>((zraw >> (8 * e)) & 255u);
      *reinterpret_cast<float2*>(table + lane * 40 + e * 8) = make_float2(v * kBack, -v * (kLeft + z));
    }
    __syncwarp();
    issue();
    if (i + 1 < mine) ask(first + (i + 1) * stride);
    float dot[2][NT][4], sx[NT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t xb[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 d = make_uint4(0u, 0u, 0u, 0u);
        if (nt * 8 + r < toks) d = lds128(stage + my_x + nt * 2048 + ((4 * j + t) ^ x_rot) * 16);
        xb[nt][0] = __byte_perm(d.x, d.z, 0x5410u), xb[nt][1] = __byte_perm(d.x, d.z, 0x7632u);
        xb[nt][2] = __byte_perm(d.y, d.w, 0x5410u), xb[nt][3] = __byte_perm(d.y, d.w, 0x7632u);
      }
      uint32_t w[4];
      ldsm4(stage + my_row + ((j ^ my_rot) << 4), w);
      const bool fresh = j % GS == 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_16816<DT>(sx[nt], ones, xb[nt][0], xb[nt][1], fresh ? none : sx[nt]);
        mma_16816<DT>(sx[nt], ones, xb[nt][2], xb[nt][3], sx[nt]);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint32_t a[2][4];  // {row r, row r + 8} x {pairs 0, 1}, {pairs 2, 3}
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e >> 1][(e & 1) * 2 + h] = ((w[2 * m + h] >> (4 * e)) & 0x000F000Fu) | kMagic;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<DT>(dot[m][nt], a[0], xb[nt][0], xb[nt][1], fresh ? none : dot[m][nt]);
          mma_16816<DT>(dot[m][nt], a[1], xb[nt][2], xb[nt][3], dot[m][nt]);
        }
      }
      if ((j + 1) % GS == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float2 lo = *reinterpret_cast<const float2*>(table + (m * 16 + r) * 40 + j / GS * 8);
          const float2 hi = *reinterpret_cast<const float2*>(table + (m * 16 + r + 8) * 40 + j / GS * 8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const Two x01 = two(sx[nt][0], sx[nt][1]);
            const float2 u = both(fma2(x01, two(lo.y), fma2(two(dot[m][nt][0], dot[m][nt][1]), two(lo.x), two(acc[m][nt][0], acc[m][nt][1]))));
            const float2 v = both(fma2(x01, two(hi.y), fma2(two(dot[m][nt][2], dot[m][nt][3]), two(hi.x), two(acc[m][nt][2], acc[m][nt][3]))));
            acc[m][nt][0] = u.x, acc[m][nt][1] = u.y, acc[m][nt][2] = v.x, acc[m][nt][3] = v.y;
          }
        }
      }
    }
    stage += S::kStep;
    if (stage == ring + S::kStages * S::kStep) stage = ring;
  }

  // Partial sums: the warps of a tile, then the CTAs of the cluster (whose tile is one).
  constexpr int TW = 8 * NT;
  cp_async_wait_all();
  __syncwarp();  // the warp is done with its ring
  float* red = reinterpret_cast<float*>(own);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[(m * 16 + (e >> 1) * 8 + r) * TW + nt * 8 + 2 * t + (e & 1)] = acc[m][nt][e];
  __syncthreads();
  auto of_tile = [&](int j, int i) {
    float v = 0.f;
    for (int w = 0; w < W; ++w) v += reinterpret_cast<const float*>(smem_w4 + (j * W + w) * S::kWarp)[i];
    return v;
  };
  float* part = reinterpret_cast<float*>(smem_w4 + kWarps * S::kWarp);
  if (Q > 1) {
    for (int i = threadIdx.x; i < kRows * TW; i += 256) part[i] = of_tile(0, i);
    cluster_sync();
  }
  const uint32_t pa = smem_u32(part);
  auto total = [&](int j, int i) {
    if (Q == 1) return of_tile(j, i);
    float v = 0.f;
    for (int c = 0; c < Q; ++c) v += ld_cluster_f32(mapa_shared(pa + i * 4, c));
    return v;
  };
  const int fold = p.joint ? 2 : 1, each = kOut * ((toks + fold - 1) / fold);
  for (int o = rank * 256 + threadIdx.x; o < per_cta * each; o += 256 * Q) {
    const int j = o / each, oo = o - j * each;
    const int tok = oo / kOut * fold, f = oo % kOut;
    const int n = (tile0 + j) * kOut + f, row = tok0 + tok;
    if (n >= p.N || row >= p.T) continue;
    float v = total(j, f * TW + tok);
    if (p.joint) v += total(j, f * TW + tok + 1);
    if constexpr (GATED) v = both(gate_act(p.act, two(v))).x * total(j, (16 + f) * TW + tok);
    else if (p.bias != nullptr) v += load_vec(p.bias, DT, n);
    const uint32_t hi = pack2<DT>(v, 0.f);
    unsigned short* out = static_cast<unsigned short*>(p.out) + (p.split ? 2 * row : p.joint ? row / 2 : row) * p.ldo + n;
    *out = static_cast<unsigned short>(hi);
    if (p.split) out[p.ldo] = static_cast<unsigned short>(pack2<DT>(v - unpack2<DT>(hi).x, 0.f));
  }
  if (Q > 1) cluster_sync();  // the others may still read this CTA's sums
}

// ---------------------------------------------------------------------- host
template <bool GATED, int NT, int XT, int GS, int DT>
cudaError_t launch(W4Params p, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0};
  constexpr int kOut = GATED ? 16 : 32;
  const long long tiles = (p.N + kOut - 1) / kOut;
  const int chunks = (p.T + 8 * NT - 1) / (8 * NT), steps = (p.K + 127) / 128;
  // About as many warps as fit at once; a warp keeps a step or more.
  const long long fit = 7ll * W4Shape<NT, XT>::kCtas * sms;
  int W = 1, Q = 1;
  while (W < kWarps && tiles * chunks * W < fit && steps >= 2 * W) W *= 2;
  while (W == kWarps && Q < 8 && tiles * chunks * Q * W < 8ll * sms && steps >= kWarps * Q * 2) Q *= 2;
  p.share = W;
  const long long ctas = (tiles + kWarps / W - 1) / (kWarps / W) * Q;
  return launch_pdl(fo_w4_kernel<GATED, NT, XT, GS, DT>, opted, dim3(static_cast<unsigned>(ctas), chunks), dim3(256), W4Shape<NT, XT>::kSmem,
                    Q, stream, p);
}

template <bool GATED, int GS, int DT>
cudaError_t by_tokens(const W4Params& p, int sms, cudaStream_t s) {
  if (p.T <= 2) return launch<GATED, 1, 2, GS, DT>(p, sms, s);
  if (p.T <= 8) return launch<GATED, 1, 8, GS, DT>(p, sms, s);
  if (p.T <= 16) return launch<GATED, 2, 16, GS, DT>(p, sms, s);
  return launch<GATED, 4, 32, GS, DT>(p, sms, s);
}

template <bool GATED, int DT>
cudaError_t by_group(const W4Params& p, int sms, cudaStream_t s) {
  if (p.per32 % 4 == 0) return by_tokens<GATED, 4, DT>(p, sms, s);
  if (p.per32 == 2) return by_tokens<GATED, 2, DT>(p, sms, s);
  return by_tokens<GATED, 1, DT>(p, sms, s);
}

int check_weight(const FoW4* w, int64_t K, const char* name) {
  if (w->q == nullptr || w->scales == nullptr || !host_aligned16(w->q))
    return host_fail(FO_EINVAL, "%s: q and scales must be device pointers, q 16-byte aligned", name);
  if (w->group <= 0 || w->group % 32 != 0) return host_fail(FO_EINVAL, "%s: group must be a positive multiple of 32, got %d", name, w->group);
  const int64_t groups = (K + w->group - 1) / w->group;
  if (w->ldq < K / 2 || w->ldq % 16 != 0)
    return host_fail(FO_EINVAL, "%s: ldq must be a multiple of 16 bytes and >= K / 2, got %lld", name, static_cast<long long>(w->ldq));
  if (w->lds < groups || (w->zeros != nullptr && w->ldz < groups))
    return host_fail(FO_EINVAL, "%s: rows of scales or zeros are shorter than the %lld groups", name, static_cast<long long>(groups));
  return FO_OK;
}

void set_weight(W4Params* p, int m, const FoW4* w) {
  p->q[m] = w->q, p->ldq[m] = w->ldq;
  p->scale[m] = w->scales, p->lds[m] = w->lds;
  p->zero[m] = static_cast<const unsigned char*>(w->zeros), p->ldz[m] = w->ldz;
}

}  // namespace
}  // namespace fo

namespace fo {
namespace {

int check_sizes(int64_t T, int64_t N, int64_t K, int dtype) {
  if (T < 0 || N < 0 || K < 0) return host_fail(FO_EINVAL, "negative problem size");
  if (T > (1ll << 19) || N > (1ll << 27) || K > (1ll << 27)) return host_fail(FO_EINVAL, "problem too large");
  if (dtype != FO_DT_F16 && dtype != FO_DT_BF16) return host_fail(FO_EINVAL, "dtype must be FO_DT_F16 or FO_DT_BF16");
  if (K % 32 != 0) return host_fail(FO_EINVAL, "4-bit rows hold whole 16-byte blocks of 32 weights: K = %lld", static_cast<long long>(K));
  return FO_OK;
}

int check_x(const void* x, int64_t ldx, int64_t T, int64_t K) {
  if (x == nullptr || !host_aligned16(x)) return host_fail(FO_EINVAL, "x must be a 16-byte aligned device pointer");
  if (ldx % 8 != 0 || (T > 1 && ldx < K))
    return host_fail(FO_EINVAL, "the row stride of x must be a multiple of 8 and >= %lld", static_cast<long long>(K));
  return FO_OK;
}

int act_code(int act) {
  switch (act) {
    case FO_GATE_SILU: return ACT_SILU;
    case FO_GATE_GELU_TANH: return ACT_GELU_TANH;
    case FO_GATE_GELU_ERF: return ACT_GELU_ERF;
    default: return ACT_RELU;
  }
}

int run(W4Params p, bool gated, int dtype, const HostDevice& hd, cudaStream_t st) {
  const uint32_t per = static_cast<uint32_t>(p.per32) / 4;  // steps a group
  p.rcp = per > 1 ? static_cast<uint32_t>((0x100000000ull + per - 1) / per) : 0u;
  p.vec = p.per32 == 1;
  for (int m = 0; m < (gated ? 2 : 1); ++m)
    p.vec = p.vec && p.lds[m] % 4 == 0 && reinterpret_cast<uintptr_t>(p.scale[m]) % 8 == 0 &&
            (p.zero[m] == nullptr || (p.ldz[m] % 4 == 0 && reinterpret_cast<uintptr_t>(p.zero[m]) % 4 == 0));
  const bool bf = dtype == FO_DT_BF16;
  const cudaError_t e = gated ? (bf ? by_group<true, DT_BF16>(p, hd.sms, st) : by_group<true, DT_F16>(p, hd.sms, st))
                              : (bf ? by_group<false, DT_BF16>(p, hd.sms, st) : by_group<false, DT_F16>(p, hd.sms, st));
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(1);
  return FO_OK;
}

}  // namespace
}  // namespace fo

extern "C" int fo_matvec_w4(const FoMatvecW4Desc* d, void* stream) {
  using namespace fo;
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (int rc = check_sizes(d->T, d->N, d->K, d->dtype)) return rc;
  if (d->T == 0 || d->N == 0) return host_ok();
  if (d->K == 0) return host_fail(FO_EINVAL, "K must be positive");
  if (int rc = check_weight(&d->w, d->K, "w")) return rc;
  if (int rc = check_x(d->x, d->ldx, d->T, d->K)) return rc;
  if (d->out == nullptr || d->ldo < d->N) return host_fail(FO_EINVAL, "out must be a device pointer with rows of N values or more");
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  W4Params p = {};
  p.x = d->x, p.ldx = d->ldx, p.T = static_cast<int>(d->T), p.N = static_cast<int>(d->N), p.K = static_cast<int>(d->K);
  set_weight(&p, 0, &d->w);
  p.per32 = d->w.group / 32;
  p.bias = d->bias, p.out = d->out, p.ldo = d->ldo;
  if (int rc = run(p, false, d->dtype, hd, static_cast<cudaStream_t>(stream))) return rc;
  return host_ok();
}

extern "C" size_t fo_gated_ffn_w4_workspace_size(const FoGatedFfnW4Desc* d) {
  if (d == nullptr || d->T <= 0 || d->F <= 0) return 0;
  return static_cast<size_t>(d->T) * 2 * ((d->F + 7) / 8 * 8) * 2;
}

extern "C" int fo_gated_ffn_w4(const FoGatedFfnW4Desc* d, void* stream) {
  using namespace fo;
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (int rc = check_sizes(d->T, d->F, d->D, d->dtype)) return rc;
  if (int rc = check_sizes(2 * d->T, d->N, d->F, d->dtype)) return rc;
  if (d->act < FO_GATE_SILU || d->act > FO_GATE_RELU) return host_fail(FO_EINVAL, "bad activation %d", d->act);
  if (d->T == 0 || d->N == 0) return host_ok();
  if (d->D == 0 || d->F == 0) return host_fail(FO_EINVAL, "D and F must be positive");
  if (int rc = check_weight(&d->w_gate, d->D, "w_gate")) return rc;
  if (int rc = check_weight(&d->w_up, d->D, "w_up")) return rc;
  if (int rc = check_weight(&d->w_down, d->F, "w_down")) return rc;
  if (d->w_gate.group != d->w_up.group) return host_fail(FO_EINVAL, "w_gate and w_up must share the group size");
  if (int rc = check_x(d->x, d->ldx, d->T, d->D)) return rc;
  if (d->out == nullptr || d->ldo < d->N) return host_fail(FO_EINVAL, "out must be a device pointer with rows of N values or more");
  const size_t need = fo_gated_ffn_w4_workspace_size(d);
  if (d->workspace == nullptr || d->workspace_bytes < need || !host_aligned16(d->workspace))
    return host_fail(FO_EINVAL, "the block needs a 16-byte aligned workspace of %zu bytes", need);
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  W4Params p = {};
  p.x = d->x, p.ldx = d->ldx, p.T = static_cast<int>(d->T), p.N = static_cast<int>(d->F), p.K = static_cast<int>(d->D);
  set_weight(&p, 0, &d->w_gate);
  set_weight(&p, 1, &d->w_up);
  p.per32 = d->w_gate.group / 32;
  p.act = act_code(d->act);
  p.out = d->workspace, p.ldo = (d->F + 7) / 8 * 8;
  p.split = 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = run(p, true, d->dtype, hd, st)) return rc;
  W4Params o = {};
  o.x = d->workspace, o.ldx = p.ldo, o.T = 2 * p.T, o.N = static_cast<int>(d->N), o.K = p.N;
  set_weight(&o, 0, &d->w_down);
  o.per32 = d->w_down.group / 32;
  o.out = d->out, o.ldo = d->ldo;
  o.joint = 1;
  if (int rc = run(o, false, d->dtype, hd, st)) return rc;
  return host_ok();
}
