// fo_skinny.cuh -- products of a few tokens with a weight matrix, out[t, n] = sum_k x[t, k]
// w[n, k]: weights of 16 bits ([N, K] or [K, N]) or of 4 bits with group scales, plain
// (optional bias) or gated, act(x Wg^T) * (x Wu^T).
//
// Bound by the weights' bytes: each is read once, by 16-byte cp.async into a ring that every
// warp keeps for itself (no block-wide barrier in the loop), straight into the fragments of
// mma.m16n8k16, whose 16 rows are weight rows and whose 8 columns are tokens, so up to 8
// tokens cost what one costs.  The K order inside a step is free as long as both operands
// share it; each layout takes the order that needs no exchange between lanes:
//   [N, K] 16 bit   a lane's 16 bytes are 8 consecutive k of its row: two MMAs
//   [K, N] 16 bit   a lane holds 8 columns of 4 consecutive k; byte permutes pair the k's,
//                   eight MMAs take one column each
//   4 bit           a 32-bit word holds 8 consecutive k; its nibbles pair as (0,4), (1,5),
//                   (2,6), (3,7), turned into exact integers q - zero by one logic operation
//                   (the bits of 1024 + q, or 128 + q in bf16) and one subtraction a pair;
//                   the group's sum is scaled in fp32
// The 8 warps of a CTA and the CTAs of a cluster split K; partial sums meet in shared
// memory (distributed across the cluster) and are added in a fixed order.
#pragma once
#include "fo_math.cuh"

namespace fo {

enum : int { W_NK = 0, W_KN = 1, W_Q4 = 2 };

struct SkinnyParams {
  const void* x;
  long long ldx;
  int T, N, K;
  const void* w[2];   // [1]: the up weights of a gated product
  long long ldw[2];   // elements; bytes for 4 bit
  const void* scale[2];
  const unsigned char* zero[2];  // null: 8
  long long lds[2], ldz[2];
  int group, groups;
  int scale_vec, zero_vec;  // their rows are read by 16 bytes
  const void* bias;
  int act;
  void *out, *g, *u;  // g, u: the products before the activation (or null)
  long long ldo, ldg, ldu;
  int early_w;  // the weights are final before the previous kernel ends: prefetch them
};

template <int DT>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (DT == DT_BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// The four pairs (k, k + 4) of a word's nibbles, minus `zero` (both halves): exact.
template <int DT>
__device__ __forceinline__ void open_q4(uint32_t w, uint32_t zero, uint32_t (&out)[4]) {
  constexpr uint32_t magic = DT == DT_BF16 ? 0x43004300u : 0x64006400u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | magic;
    if constexpr (DT == DT_BF16) {
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&zero));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    } else {
      const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&zero));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

template <int FMT, bool GATED>
struct SkinnyShape {
  static constexpr int kWarps = 8;
  static constexpr int kStep = FMT == W_KN ? 16 : FMT == W_Q4 ? 128 : 32;  // k of a warp's step
  static constexpr int kChunks = FMT == W_KN ? 8 : (GATED ? 4 : 2);        // 16-byte loads a lane and step
  static constexpr int kStages = FMT == W_KN ? 3 : (GATED ? 4 : 6);
  static constexpr int kFeatures = FMT == W_KN ? (GATED ? 64 : 128) : 16;  // outputs of a CTA
  static constexpr int kRows = GATED ? 2 * kFeatures : kFeatures;          // weight rows of a CTA
  static constexpr int kTiles = FMT == W_KN ? 8 : (GATED ? 2 : 1);         // 16-row MMA tiles of a warp
  static constexpr int ring_bytes() { return kWarps * kStages * kChunks * 512; }
  static constexpr int red_bytes(int nt) { return kWarps * kRows * 8 * nt * 4; }
  static constexpr int main_bytes(int nt) { return ring_bytes() > red_bytes(nt) ? ring_bytes() : red_bytes(nt); }
  static constexpr int part_bytes(int nt) { return kRows * 8 * nt * 4; }
  // rows of scales and zeros start 16 bytes further round the banks than the row before
  static constexpr int scale_stride(int groups) { return (groups * 2 + 15) / 16 * 16 + 16; }
  static constexpr int zero_stride(int groups) { return (groups + 15) / 16 * 16 + 16; }
  static constexpr int smem_bytes(int nt, int groups, bool zeros) {
    return main_bytes(nt) + part_bytes(nt) +
           (FMT == W_Q4 ? kRows * (scale_stride(groups) + (zeros ? zero_stride(groups) : 0)) : 0);
  }
};

template <int FMT, bool GATED, int NT, int DT>
__global__ void __launch_bounds__(256) fo_skinny_kernel(const SkinnyParams p) {
  using S = SkinnyShape<FMT, GATED>;
  extern __shared__ __align__(128) uint8_t smem_sk[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  int q, Q;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(q));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(Q));
  const int n0 = static_cast<int>(blockIdx.x / Q) * S::kFeatures;
  const int tok0 = static_cast<int>(blockIdx.y) * 8 * NT;
  const int steps = (p.K + S::kStep - 1) / S::kStep;
  const int first = q * S::kWarps + warp, stride = Q * S::kWarps;
  const int mine = first < steps ? (steps - first + stride - 1) / stride : 0;
  const uint32_t ring = smem_u32(smem_sk) + warp * (S::kStages * S::kChunks * 512);
  float* part = reinterpret_cast<float*>(smem_sk + S::main_bytes(NT));
  uint8_t* scales = smem_sk + S::main_bytes(NT) + S::part_bytes(NT);
  const int sstride = S::scale_stride(p.groups), zstride = S::zero_stride(p.groups);
  uint8_t* zeros = scales + S::kRows * sstride;

  auto issue = [&](int i) {  // this warp's i-th step into its ring (an empty group past the end)
    if (i < mine) {
      const int s = first + i * stride;
      const uint32_t dst = ring + (i % S::kStages) * (S::kChunks * 512);
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        const char* base = static_cast<const char*>(p.w[0]);
        const char* src;
        bool in;
        uint32_t at = lane * 16;
        if constexpr (FMT == W_KN) {
          const int m = GATED ? c >> 2 : 0;
          const int k = s * 16 + 4 * t + (c & 3), n = n0 + (GATED ? 0 : (c >> 2) * 64) + r * 8;
          base = static_cast<const char*>(p.w[m]);
          in = k < p.K && n < p.N;
          src = base + (static_cast<long long>(k) * p.ldw[m] + n) * 2;
        } else {
          const int m = c >> 1;
          const int n = n0 + r + 8 * (c & 1);
          base = static_cast<const char*>(p.w[m]);
          if constexpr (FMT == W_NK) {
            const int k = s * 32 + t * 8;
            in = n < p.N && k < p.K;
            src = base + (static_cast<long long>(n) * p.ldw[m] + k) * 2;
          } else {
            in = n < p.N && s * 128 + t * 32 < p.K;
            src = base + static_cast<long long>(n) * p.ldw[m] + s * 64 + t * 16;
            at = (r * 4 + (t ^ ((r >> 1) & 3))) * 16;  // any 4-byte column of the 8 rows: distinct banks
          }
        }
        cp_async_16(dst + c * 512 + at, in ? src : base, in ? 16u : 0u);
      }
    }
    cp_async_commit();
  };

  griddep_wait();
  griddep_launch_dependents();
  if constexpr (FMT == W_Q4) {
    // The rows' scales and zeros, whole: a warp takes rows warp, warp + 8, .. by 16-byte
    // copies where the rows allow them (they land with the ring's first steps), else by
    // single loads.
    for (int row = warp; row < S::kRows; row += S::kWarps) {
      const int m = row / S::kFeatures, n = n0 + row % S::kFeatures;
      const bool in = n < p.N;
      const unsigned short* sc = static_cast<const unsigned short*>(p.scale[m]) + (in ? n : 0) * p.lds[m];
      unsigned short* sd = reinterpret_cast<unsigned short*>(scales + row * sstride);
      if (p.scale_vec) {
        for (int i = lane * 8; i < p.groups; i += 256) cp_async_16(smem_u32(sd + i), sc + i, in ? 16u : 0u);
      } else {
        for (int i = lane; i < p.groups; i += 32) sd[i] = in ? __ldg(sc + i) : 0;
      }
      if (p.zero[0] != nullptr) {
        const unsigned char* zc = p.zero[m] + (in ? n : 0) * p.ldz[m];
        unsigned char* zd = zeros + row * zstride;
        if (p.zero_vec) {
          for (int i = lane * 16; i < p.groups; i += 512) cp_async_16(smem_u32(zd + i), zc + i, in ? 16u : 0u);
        } else {
          for (int i = lane; i < p.groups; i += 32) zd[i] = in ? __ldg(zc + i) : 0;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);
  if constexpr (FMT == W_Q4) {
    cp_async_wait<S::kStages - 2>();  // the scales are older than every step but the first, and land with it
    __syncthreads();
  }

  float acc[S::kTiles][NT][4] = {};
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<S::kStages - 2>();
    if constexpr (FMT == W_Q4) __syncwarp();  // other lanes' copies, and their reads of the slot refilled next
    issue(i + S::kStages - 1);
    const int s = first + i * stride;
    const uint32_t src = ring + (i % S::kStages) * (S::kChunks * 512);
    const unsigned short* xp = static_cast<const unsigned short*>(p.x);
    if constexpr (FMT == W_NK) {
      uint4 xf[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int tok = tok0 + nt * 8 + r, k = s * 32 + t * 8;
        xf[nt] = make_uint4(0u, 0u, 0u, 0u);
        if (tok < p.T && k < p.K) xf[nt] = __ldg(reinterpret_cast<const uint4*>(xp + tok * p.ldx + k));
      }
#pragma unroll
      for (int m = 0; m < S::kTiles; ++m) {
        const uint4 lo = lds128(src + (2 * m) * 512 + lane * 16), hi = lds128(src + (2 * m + 1) * 512 + lane * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<DT>(acc[m][nt], lo.x, hi.x, lo.y, hi.y, xf[nt].x, xf[nt].y);
          mma_16816<DT>(acc[m][nt], lo.z, hi.z, lo.w, hi.w, xf[nt].z, xf[nt].w);
        }
      }
    } else if constexpr (FMT == W_KN) {
      uint2 xf[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int tok = tok0 + nt * 8 + r, k = s * 16 + 4 * t;
        xf[nt] = make_uint2(0u, 0u);
        if (tok < p.T && k < p.K) xf[nt] = __ldg(reinterpret_cast<const uint2*>(xp + tok * p.ldx + k));
      }
      uint32_t v[8][4];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 d = lds128(src + c * 512 + lane * 16);
        v[c][0] = d.x, v[c][1] = d.y, v[c][2] = d.z, v[c][3] = d.w;
      }
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const uint32_t sel = (m & 1) ? 0x7632u : 0x5410u;
        const int e = m >> 1;
        const uint32_t a0 = __byte_perm(v[0][e], v[1][e], sel), a2 = __byte_perm(v[2][e], v[3][e], sel);
        const uint32_t a1 = __byte_perm(v[4][e], v[5][e], sel), a3 = __byte_perm(v[6][e], v[7][e], sel);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816<DT>(acc[m][nt], a0, a1, a2, a3, xf[nt].x, xf[nt].y);
      }
    } else {
      float ag[S::kTiles][NT][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k0 = s * 128 + j * 32;
        if (k0 >= p.K) break;
        const int gi = k0 / p.group;
        if (j == 0 || k0 % p.group == 0) {
#pragma unroll
          for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) ag[m][nt][e] = 0.f;
        }
        uint32_t xb[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int tok = tok0 + nt * 8 + r;
          uint4 d = make_uint4(0u, 0u, 0u, 0u);
          if (tok < p.T) d = __ldg(reinterpret_cast<const uint4*>(xp + tok * p.ldx + k0 + 8 * t));
          xb[nt][0] = __byte_perm(d.x, d.z, 0x5410u), xb[nt][1] = __byte_perm(d.x, d.z, 0x7632u);
          xb[nt][2] = __byte_perm(d.y, d.w, 0x5410u), xb[nt][3] = __byte_perm(d.y, d.w, 0x7632u);
        }
        const uint32_t at = (r * 4 + (j ^ ((r >> 1) & 3))) * 16 + t * 4;
#pragma unroll
        for (int m = 0; m < S::kTiles; ++m) {
          uint32_t z[2] = {8u, 8u};
          if (p.zero[0] != nullptr) {
            z[0] = zeros[(m * 16 + r) * zstride + gi];
            z[1] = zeros[(m * 16 + r + 8) * zstride + gi];
          }
          uint32_t lo[4], hi[4];
          constexpr uint32_t magic = DT == DT_BF16 ? 0x4300u : 0x6400u;
          open_q4<DT>(lds32(src + (2 * m) * 512 + at), (magic | z[0]) * 0x10001u, lo);
          open_q4<DT>(lds32(src + (2 * m + 1) * 512 + at), (magic | z[1]) * 0x10001u, hi);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816<DT>(ag[m][nt], lo[0], hi[0], lo[1], hi[1], xb[nt][0], xb[nt][1]);
            mma_16816<DT>(ag[m][nt], lo[2], hi[2], lo[3], hi[3], xb[nt][2], xb[nt][3]);
          }
        }
        if (j == 3 || (k0 + 32) % p.group == 0 || k0 + 32 >= p.K) {
#pragma unroll
          for (int m = 0; m < S::kTiles; ++m) {
            const float s0 = unpack2<DT>(*reinterpret_cast<const unsigned short*>(scales + (m * 16 + r) * sstride + gi * 2)).x;
            const float s1 = unpack2<DT>(*reinterpret_cast<const unsigned short*>(scales + (m * 16 + r + 8) * sstride + gi * 2)).x;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[m][nt][0] = fmaf(ag[m][nt][0], s0, acc[m][nt][0]);
              acc[m][nt][1] = fmaf(ag[m][nt][1], s0, acc[m][nt][1]);
              acc[m][nt][2] = fmaf(ag[m][nt][2], s1, acc[m][nt][2]);
              acc[m][nt][3] = fmaf(ag[m][nt][3], s1, acc[m][nt][3]);
            }
          }
        }
      }
    }
  }

  // Partial sums: warps of the CTA, then CTAs of the cluster.
  constexpr int TW = 8 * NT;
  cp_async_wait_all();
  __syncthreads();  // every warp is done with its ring
  float* red = reinterpret_cast<float*>(smem_sk) + warp * S::kRows * TW;
#pragma unroll
  for (int m = 0; m < S::kTiles; ++m)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // a tile's rows: 16 weight rows, or in the [K, N] layout column m of the 8 (of each half)
        const int hi = e >> 1;
        const int row = FMT == W_KN ? hi * 64 + r * 8 + m : m * 16 + hi * 8 + r;
        red[row * TW + nt * 8 + 2 * t + (e & 1)] = acc[m][nt][e];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < S::kRows * TW; i += 256) {
    const float* s0 = reinterpret_cast<const float*>(smem_sk) + i;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) v += s0[w * S::kRows * TW];
    part[i] = v;
  }
  if (Q > 1) cluster_sync(); else __syncthreads();
  const uint32_t pa = smem_u32(part);
  auto total = [&](int i) {
    if (Q == 1) return part[i];
    float v = 0.f;
    for (int c = 0; c < Q; ++c) v += ld_cluster_f32(mapa_shared(pa + i * 4, c));
    return v;
  };
  for (int o = q * 256 + threadIdx.x; o < S::kFeatures * TW; o += 256 * Q) {
    const int tok = o / S::kFeatures, f = o - tok * S::kFeatures;
    const int n = n0 + f, row = tok0 + tok;
    if (n >= p.N || row >= p.T) continue;
    float v = total(f * TW + tok);
    if constexpr (GATED) {
      const float u = total((S::kFeatures + f) * TW + tok);
      if (p.g != nullptr) {
        static_cast<unsigned short*>(p.g)[row * p.ldg + n] = static_cast<unsigned short>(pack2<DT>(v, 0.f));
        static_cast<unsigned short*>(p.u)[row * p.ldu + n] = static_cast<unsigned short>(pack2<DT>(u, 0.f));
      }
      v = both(gate_act(p.act, two(v))).x * u;
    } else if (p.bias != nullptr) {
      v += load_vec(p.bias, DT, n);
    }
    static_cast<unsigned short*>(p.out)[row * p.ldo + n] = static_cast<unsigned short>(pack2<DT>(v, 0.f));
  }
  if (Q > 1) cluster_sync();  // the others may still read this CTA's sums
}

// Launches the product (host); FMT, GATED and the dtype are those of the call.
int gate_act_of(int act);  // FO_GATE_* -> ACT_*
cudaError_t launch_skinny(int fmt, bool gated, int dt, const SkinnyParams& p, int sms, cudaStream_t stream);

}  // namespace fo
