// fo_few.cuh -- the tcgen05 kernel for products whose token side is short: the weights are
// the MMA's M side (128 features a tile), the tokens its N side (NT = 16, 32 or, but for
// FEW_GATED, 64 columns, all of them in one tile).
//
// With few tokens the time is that of the weights' bytes: an MMA costs by its token columns,
// so nothing is spent on absent rows, and a SM keeps about 200 KB of weight tiles in flight
// (two CTAs a SM where their rings fit).  Where the tiles are fewer than the SMs, the Q CTAs
// of a cluster take a tile's K blocks together: each pushes its sums of the token columns it
// does not own into their owner's shared memory, and the owner adds them in rank order
// (fixed, so results do not depend on timing) and runs the epilogue.
//
// The accumulator's lanes are features and its columns tokens, so a gated product's g and u
// of one value lie in one lane, and a warp writes 64 contiguous bytes a token.
//   FEW_GATED  two weight tiles a K block: h = act(g) * u (and g, u)
//   FEW_PLAIN  one weight tile a K block, over one or two K segments
//   FEW_DGATE  FEW_PLAIN's accumulator is dh: writes dg, du, h from the saved g, u
// Between the forward pass's two products h travels as two 16-bit parts, high and low, in rows
// 2 t and 2 t + 1: twice the token columns of an MMA that is not the bound, and h keeps 16
// significant bits in bf16, 22 in fp16 (there down to steps of 2^-24).
//
// Measured, both products of the block, bf16: 4096 x 16384, 403 MB, one token in 66 us (6.1
// TB/s), 24 tokens in 78 us; 1 x 1024 x 4096, 25 MB in 12.7 us (10.9 from L2), bound by the
// launches and the first copies' latency.
#pragma once
#include "fo_ffn.cuh"

namespace fo {

enum : int { FEW_GATED = 0, FEW_PLAIN = 1, FEW_DGATE = 2 };

constexpr int kFewThreads = 192;
constexpr int kFewMaxStages = 8;

template <int MODE, int NT>
struct FewShape {
  static constexpr int kTiles = MODE == FEW_GATED ? 2 : 1;      // weight tiles a K block
  static constexpr int kW = kTiles * kAStageBytes;              // weight bytes a stage (one K block)
  static constexpr int kStage = kW + NT * kBK * 2;
  static constexpr int kCols = NT < 32 ? 32 : NT;               // TMEM columns of one product
  static constexpr int kTmem = kTiles * kCols;
  static constexpr int kExchange = kTiles * NT * 128 * 4;       // sums received from the cluster
  static constexpr int kBudget = 110 * 1024;                    // two CTAs a SM
  static constexpr int kStages = kBudget / kStage < kFewMaxStages ? kBudget / kStage : kFewMaxStages;
  static constexpr int kRing = kStages * kStage > kExchange ? kStages * kStage : kExchange;
  static constexpr int kSmem = 1024 + kRing + 512;
  static_assert(kStages >= 2, "a ring");
};

struct FewMaps {
  CUtensorMap a[2], b[2];  // weights (gate, up; or the K segments'), tokens (the segments')
};

struct FewParams {
  int F, T;             // features, token columns (two a token where joint)
  int kb0, kb;          // K blocks of the first segment, of all
  int a_mn, bf16;
  void *out, *g, *u;    // FEW_GATED: h, g, u (or null); FEW_PLAIN: out; FEW_DGATE: dg, du, h
  long long ldo, ldg, ldu;
  const void *sg, *su;  // FEW_DGATE: the saved g, u
  long long ldsg, ldsu;
  int split, joint;     // FEW_GATED: h is written in two parts; FEW_PLAIN: it comes so
  int early;            // the weights are final before the previous kernel ends
  int* status;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ void few_error(const FewParams& p, int where) {
  if (atomicCAS(p.status, 0, kStatusTimeout) == 0) {
    p.status[1] = where;
    p.status[2] = static_cast<int>(blockIdx.x);
  }
}

__device__ __forceinline__ unsigned short to16(float v, int bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ float from16(unsigned short v, int bf16) {
  return bf16 ? __bfloat162float(__ushort_as_bfloat16(v)) : __half2float(__ushort_as_half(v));
}

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int MODE, int ACT, int NT>
__global__ void __launch_bounds__(kFewThreads) fo_few_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewParams p) {
  using S = FewShape<MODE, NT>;
  extern __shared__ __align__(1024) uint8_t smem_few[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_few) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t ring = smem_u32(smem);
  uint8_t* misc = smem + S::kRing;
  const uint32_t mb = smem_u32(misc);
  const uint32_t bar_full = mb, bar_empty = mb + 64, bar_tfull = mb + 128;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 248);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 252);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int Q;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(Q));
  const int rank = static_cast<int>(cluster_ctarank());
  const int f0 = static_cast<int>(blockIdx.x) / Q * 128;
  const int k0 = p.kb * rank / Q, k1 = p.kb * (rank + 1) / Q;  // this CTA's K blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), S::kTmem);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint64_t tmo = p.timeout_ns;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      auto weights = [&](int kb, int s) {
        const uint32_t fb = bar_full + 8 * s, w = ring + s * S::kStage;
        mbar_arrive_expect_tx(fb, S::kStage);
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
          const int seg = MODE == FEW_GATED ? i : kb >= p.kb0;
          const int k = (kb - (MODE != FEW_GATED && seg ? p.kb0 : 0)) * kBK;
          if (p.a_mn) {
            tma_load_2d(w + i * kAStageBytes, &maps.a[seg], fb, f0, k);
            tma_load_2d(w + i * kAStageBytes + 64 * 128, &maps.a[seg], fb, f0 + 64, k);
          } else {
            tma_load_2d(w + i * kAStageBytes, &maps.a[seg], fb, k, f0);
          }
        }
      };
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      int ahead = k0;  // weight stages asked for before the tokens exist
      if (p.early)
        for (; ahead < k1 && ahead - k0 < S::kStages; ++ahead) weights(ahead, ahead - k0);
      griddep_wait();
      for (int kb = k0; kb < k1; ++kb) {
        if (kb >= ahead) {
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, tmo, abort_flag)) {
            ok = false;
            break;
          }
          weights(kb, s);
        }
        const int seg = MODE != FEW_GATED && kb >= p.kb0;
        tma_load_2d(ring + s * S::kStage + S::kW, &maps.b[seg], bar_full + 8 * s, (kb - (seg ? p.kb0 : 0)) * kBK, 0);
        ++issued;
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) {
        few_error(p, 0x60);
        *abort_flag = 1;
      }
      drain_loads(bar_full, S::kStages, issued);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc = idesc_f16(p.bf16, 0, NT, 128) | (static_cast<uint32_t>(p.a_mn) << 15);
      const uint64_t a0 = p.a_mn ? sdesc_sw128(ring, 64 * 128, 1024) : sdesc_sw128(ring, 16, 1024);
      const uint64_t b0 = sdesc_sw128(ring + S::kW, 16, 1024);
      const uint32_t as = p.a_mn ? (2048 >> 4) : (32 >> 4), bs = 32 >> 4;
      int s = 0;
      uint32_t ph = 0, accum = 0;
      bool ok = true;
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(bar_full + 8 * s, ph, tmo, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t off = static_cast<uint64_t>(s * (S::kStage >> 4));
#pragma unroll
        for (int i = 0; i < S::kTiles; ++i) {
          const uint64_t a = a0 + off + i * (kAStageBytes >> 4), b = b0 + off;
          const uint32_t d = tmem_base + i * S::kCols;
          tc_mma_f16(d, a, b, idesc, accum);
          tc_mma_f16(d, a + as, b + bs, idesc, 1u);
          tc_mma_f16(d, a + 2 * as, b + 2 * bs, idesc, 1u);
          tc_mma_f16(d, a + 3 * as, b + 3 * bs, idesc, 1u);
        }
        accum = 1u;
        tc_commit(bar_empty + 8 * s);
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) {
        few_error(p, 0x61);
        *abort_flag = 1;
      }
      tc_commit(bar_tfull);  // every MMA issued has completed
      mbar_wait(bar_tfull, 0, kDrainTimeoutNs, nullptr);
    }
  } else {
    // Everything before this kernel has completed: the next one may start its setup.
    griddep_wait();
    griddep_launch_dependents();
    if (!mbar_wait(bar_tfull, 0, tmo, abort_flag) && lane == 0) {
      few_error(p, 0x62);
      *abort_flag = 1;
    }
  }
  __syncwarp();

  const int quarter = warp & 3;
  const uint32_t tb = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  const int f = f0 + quarter * 32 + lane;
  auto finish = [&](int t, float v, float w) {
    if (f >= p.F || t >= p.T) return;
    unsigned short* out = static_cast<unsigned short*>(p.out) + (MODE == FEW_GATED && p.split ? 2 * t : MODE == FEW_PLAIN && p.joint ? t / 2 : t) * p.ldo + f;
    if constexpr (MODE == FEW_GATED) {
      if (p.g != nullptr) {
        static_cast<unsigned short*>(p.g)[t * p.ldg + f] = to16(v, p.bf16);
        static_cast<unsigned short*>(p.u)[t * p.ldu + f] = to16(w, p.bf16);
      }
      const float h = both(gate_act<ACT>(two(v))).x * w;
      const unsigned short hi = to16(h, p.bf16);
      *out = hi;
      if (p.split) out[p.ldo] = to16(low_part(h, from16(hi, p.bf16)), p.bf16);
    } else if constexpr (MODE == FEW_DGATE) {
      const float sg = from16(__ldg(static_cast<const unsigned short*>(p.sg) + t * p.ldsg + f), p.bf16);
      const float su = from16(__ldg(static_cast<const unsigned short*>(p.su) + t * p.ldsu + f), p.bf16);
      Two dg, du, h;
      gate_grad<ACT>(two(v), two(sg), two(su), dg, du, h);
      *out = to16(both(dg).x, p.bf16);
      static_cast<unsigned short*>(p.g)[t * p.ldg + f] = to16(both(du).x, p.bf16);
      static_cast<unsigned short*>(p.u)[t * p.ldu + f] = to16(both(h).x, p.bf16);
    } else {
      *out = to16(v, p.bf16);
    }
  };
  constexpr int kChunk = NT < 32 ? NT : 32;
  if (Q == 1) {
    if (warp >= 2) {
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < NT && c0 < p.T; c0 += kChunk) {
        uint32_t r[32], s[32];
        tmem_ld_32x32b_x32(tb + c0, r);
        if constexpr (MODE == FEW_GATED) tmem_ld_32x32b_x32(tb + S::kCols + c0, s);
        tc_wait_ld_regs(r);
        if constexpr (MODE == FEW_GATED) tc_pin_regs(s);
        if (MODE == FEW_PLAIN && p.joint) {
#pragma unroll
          for (int i = 0; i < kChunk; i += 2) finish(c0 + i, __uint_as_float(r[i]) + __uint_as_float(r[i + 1]), 0.f);
        } else {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) finish(c0 + i, __uint_as_float(r[i]), MODE == FEW_GATED ? __uint_as_float(s[i]) : 0.f);
        }
      }
    }
  } else {
    // Rank r owns token columns r * NT / Q ..; its receive area (the idle ring) holds, for
    // each sender and product, 128 lanes of every owned column.
    const int own = NT / Q;
    cluster_sync();  // every CTA's ring is idle
    if (warp >= 2) {
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < S::kTiles * NT; c0 += kChunk) {
        const int prod = c0 / NT, j0 = c0 - prod * NT;
        uint32_t r[32];
        tmem_ld_32x32b_x32(tb + prod * S::kCols + j0, r);
        tc_wait_ld_regs(r);
        auto send = [&](int i) {
          const int j = j0 + i, to = j / own;
          st_cluster_f32(mapa_shared(ring, to) + (((rank * S::kTiles + prod) * own + j - to * own) * 128 + quarter * 32 + lane) * 4,
                         __uint_as_float(r[i]));
        };
        if (2 * (p.T - j0) > kChunk) {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) send(i);
        } else {  // few of the columns exist
#pragma unroll
          for (int i = 0; i < kChunk / 2; ++i)
            if (j0 + i < p.T) send(i);
        }
      }
    }
    cluster_sync();  // every sum has arrived
    if (warp >= 2) {
      const int step = MODE == FEW_PLAIN && p.joint ? 2 : 1;  // (own is even: NT >= 16, Q <= 8)
      for (int j = 0; j < own; j += step) {
        const int t = rank * own + j;
        if (t >= p.T) break;
        float v = 0.f, w = 0.f;
        for (int q = 0; q < Q; ++q) {
          const float* src = reinterpret_cast<const float*>(smem) + (q * S::kTiles * own + j) * 128 + quarter * 32 + lane;
          v += src[0];
          if (step == 2) w += src[128];
          if constexpr (MODE == FEW_GATED) w += src[own * 128];
        }
        if (step == 2) finish(t, v + w, 0.f);
        else finish(t, v, w);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmem);
  }
}

// Token columns, feature tiles, and the CTAs that split a tile's K blocks.
struct FewPlan {
  int nt, tiles, q;
};

FewPlan few_plan(int mode, int64_t F, int64_t columns, int kb, int sms);  // columns <= 64
cudaError_t launch_few(int mode, int act, const FewMaps& m, const FewParams& p, const FewPlan& plan, cudaStream_t stream);

}  // namespace fo
