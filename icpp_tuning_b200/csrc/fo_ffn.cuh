// fo_ffn.cuh -- the tcgen05 kernel of the gated feed-forward block's products.
//
// A persistent kernel of CTA pairs (tcgen05 cta_group::2, 256 x 256 fp32 accumulator: 128
// rows in each CTA's TMEM, two accumulators so that a tile's epilogue overlaps the next
// tile's MMAs).  Warp 0 feeds a ring of 128-byte-swizzled tiles by TMA, warp 1 of the leader
// CTA issues the MMAs, warps 2-9 run the epilogue.  Epilogues:
//   FFN_GATED  the B tile is 128 columns of Wg (loaded by CTA 0 of the pair) and the same
//              128 columns of Wu (CTA 1), so every accumulator row holds g and u of the
//              same 128 features and h = act(g) * u leaves the registers: one kernel for
//              both projections, the activation and the product (and g, u when saved)
//   FFN_DGATE  acc = dh = dy Wd^T; reads g, u and writes dg = dh u act'(g), du = dh act(g),
//              h = act(g) u: the block's whole elementwise backward, dh never in memory
//   FFN_GRADS  plain products, up to four of them in one launch, each over one or two K
//              segments with their own operands (dx = dg Wg^T + du Wu^T)
// Operands are K-major or MN-major (read transposed) per problem, so every product of the
// block and its gradients runs on tensors as they are, without a transposition pass.
#pragma once
#include "fo_skinny.cuh"

namespace fo {

enum : int { FFN_GATED = 0, FFN_DGATE = 1, FFN_GRADS = 2 };

constexpr int kFfnStages = 3;  // of two 64-wide k-blocks: 64 KB a stage and CTA
constexpr int kFfnKps = 2;
constexpr int kFfnTile = 256;  // rows and columns of a pair's accumulator
constexpr int kFfnStageA = kFfnKps * kAStageBytes, kFfnStageB = kFfnKps * 128 * kBK * 2;
constexpr int kFfnSmem = 1024 + kFfnStages * (kFfnStageA + kFfnStageB) + kEpiBytes + 512;
constexpr int kFfnMaxProblems = 4;
constexpr int kFfnOwners = 512;

struct FfnProblem {
  int M, N;
  int tiles_m, tiles_n;
  int unit0;           // first unit of this problem
  int kb0, kb;         // k-blocks of the first segment, of all
  int a_mn, b_mn;      // operands read transposed
};

struct FfnMaps {
  CUtensorMap a[kFfnMaxProblems][2], b[kFfnMaxProblems][2], c[kFfnMaxProblems];
};

struct FfnParams {
  FfnProblem prob[kFfnMaxProblems];
  int nprob, units, group_m;
  int bf16, save;
  const void *g, *u;  // FFN_DGATE
  long long ldg, ldu;
  int* status;
  unsigned long long timeout_ns;
  int owned;  // owner[u] names the pair that runs unit u (else pair u % pairs)
  unsigned char owner[kFfnOwners];
};

// dg and du of one value from dh; h too.
template <int ACT>
__device__ __forceinline__ void gate_grad(float dh, float g, float u, float& dg, float& du, float& h) {
  float s, ds;
  if constexpr (ACT == ACT_SILU) {
    const float p = sigmoid_fast(g);
    s = g * p;
    ds = fmaf(s, 1.0f - p, p);
  } else if constexpr (ACT == ACT_GELU_TANH) {
    // gelu_tanh(g) = g p, p = sigmoid(2 w), w = c (g + 0.044715 g^3): derivative p + g p (1 - p) 2 w'
    const float g2 = g * g;
    const float p = sigmoid_fast(1.5957691216057308f * fmaf(0.044715f * g, g2, g));
    s = g * p;
    ds = fmaf(s * (1.0f - p), 1.5957691216057308f * fmaf(0.134145f, g2, 1.0f), p);
  } else if constexpr (ACT == ACT_GELU_ERF) {
    const float c = 0.5f * (1.0f + erf_as7128(g * 0.7071067811865476f));
    s = g * c;
    ds = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), c);
  } else {
    s = g < 0.f ? 0.f : g;
    ds = g > 0.f ? 1.f : 0.f;
  }
  dg = dh * u * ds;
  du = dh * s;
  h = s * u;
}

__device__ __forceinline__ void ffn_error(const FfnParams& p, int where) {
  if (atomicCAS(p.status, 0, kStatusTimeout) == 0) {
    p.status[1] = where;
    p.status[2] = static_cast<int>(blockIdx.x);
  }
}

struct FfnUnit {
  int pr, tm, tn;
};

__device__ __forceinline__ FfnUnit ffn_unit(const FfnParams& p, int u) {
  FfnUnit r;
  r.pr = 0;
  while (r.pr + 1 < p.nprob && u >= p.prob[r.pr + 1].unit0) ++r.pr;
  const FfnProblem& q = p.prob[r.pr];
  const int t = u - q.unit0;
  const int per = p.group_m * q.tiles_n;  // rasters of group_m row blocks, for reuse in L2
  const int gr = t / per, in = t - gr * per;
  const int gm = min(p.group_m, q.tiles_m - gr * p.group_m);
  r.tm = gr * p.group_m + in % gm;
  r.tn = in / gm;
  return r;
}

// This pair's next unit at or after u.
__device__ __forceinline__ int ffn_next(const FfnParams& p, int u, int cid, int ncl) {
  (void)ncl;
  if (!p.owned) return u;
  while (u < p.units && p.owner[u] != cid) ++u;
  return u;
}

template <int EPI, int ACT, int DT>
__global__ void __launch_bounds__(320, 1) fo_ffn_kernel(const __grid_constant__ FfnMaps maps, const __grid_constant__ FfnParams p) {
  extern __shared__ __align__(1024) uint8_t smem_ffn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_ffn) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sA = smem_u32(smem);
  const uint32_t sB = sA + kFfnStages * kFfnStageA;
  const uint32_t sEpi = sB + kFfnStages * kFfnStageB;
  uint8_t* misc = smem + (sEpi - sA) + kEpiBytes;
  const uint32_t mb = smem_u32(misc);
  const uint32_t bar_full = mb, bar_empty = mb + 64, bar_tfull = mb + 128, bar_tempty = mb + 144, bar_drain = mb + 160;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 248);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 252);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cid = static_cast<int>(blockIdx.x >> 1), ncl = static_cast<int>(gridDim.x >> 1);
  const int step = p.owned ? 1 : ncl;       // units are walked from `first` with this step,
  const int first = p.owned ? 0 : cid;      // skipping other pairs' when owners are named

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFfnStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, 2 * kEpiWarps);
    }
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&maps.a[0][0]);
    tma_prefetch_desc(&maps.b[0][0]);
    tma_prefetch_desc(&maps.c[0]);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint64_t tmo = p.timeout_ns;
  griddep_wait();

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = ffn_next(p, first, cid, ncl); u < p.units && ok; u = ffn_next(p, u + step, cid, ncl)) {
        const FfnUnit un = ffn_unit(p, u);
        const FfnProblem& q = p.prob[un.pr];
        const int arow = un.tm * kFfnTile + static_cast<int>(rank) * 128;
        const int bcol = EPI == FFN_GATED ? un.tn * 128 : un.tn * kFfnTile + static_cast<int>(rank) * 128;
        // everything of the problem in registers: a constant read costs this one thread as
        // much as issuing a copy
        const int kb = q.kb, a_mn = q.a_mn, b_mn = q.b_mn;
        int left = q.kb0, k = 0;  // K blocks left in the segment, the next one's first column
        const CUtensorMap* ma = &maps.a[un.pr][0];
        const CUtensorMap* mB = EPI == FFN_GATED ? &maps.b[0][rank] : &maps.b[un.pr][0];
        for (int k0 = 0; k0 < kb; k0 += kFfnKps) {
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, tmo, abort_flag)) {
            ok = false;
            break;
          }
          const int nk = min(kFfnKps, kb - k0);
          const uint32_t fb = bar_full + 8 * s;
          const uint32_t fbl = mapa_shared(fb, 0);  // both CTAs' bytes complete on the leader's barrier
          if (rank == 0) mbar_arrive_expect_tx(fb, 2 * nk * (kFfnStageA + kFfnStageB) / kFfnKps);
          uint32_t sa = sA + s * kFfnStageA, sb = sB + s * kFfnStageB;
#pragma unroll
          for (int i = 0; i < kFfnKps; ++i) {
            if (i >= nk) break;
            if (EPI == FFN_GRADS && left == 0) {  // the second segment
              ++ma, ++mB;
              k = 0;
              left = kb;
            }
            if (a_mn) {
              tma_load_2d_pair(sa, ma, fbl, arow, k);
              tma_load_2d_pair(sa + 64 * 128, ma, fbl, arow + 64, k);
            } else {
              tma_load_2d_pair(sa, ma, fbl, k, arow);
            }
            if (b_mn) {
              tma_load_2d_pair(sb, mB, fbl, bcol, k);
              tma_load_2d_pair(sb + 64 * 128, mB, fbl, bcol + 64, k);
            } else {
              tma_load_2d_pair(sb, mB, fbl, k, bcol);
            }
            sa += kAStageBytes, sb += kAStageBytes;
            k += kBK;
            --left;
          }
          ++issued;
          if (++s == kFfnStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        ffn_error(p, 0x40);
        *abort_flag = 1;
      }
      if (rank == 0) drain_loads(bar_full, kFfnStages, issued);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0) {
      // One thread issues every MMA and commit: the descriptors are stepped per stage, and
      // nothing of a problem is read again inside its K loop.
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      uint64_t off = 0;  // of stage s, in descriptor units (A and B stages are alike)
      bool ok = true;
      for (int u = ffn_next(p, first, cid, ncl); u < p.units && ok; u = ffn_next(p, u + step, cid, ncl)) {
        const FfnProblem& q = p.prob[EPI == FFN_GRADS ? ffn_unit(p, u).pr : 0];
        const int kb = q.kb, a_mn = q.a_mn, b_mn = q.b_mn;
        const uint32_t idesc = idesc_f16(p.bf16, b_mn, 256, 256) | (static_cast<uint32_t>(a_mn) << 15);
        const uint64_t a0 = a_mn ? sdesc_sw128(sA, 64 * 128, 1024) : sdesc_sw128(sA, 16, 1024);
        const uint64_t b0 = b_mn ? sdesc_sw128(sB, 64 * 128, 1024) : sdesc_sw128(sB, 16, 1024);
        const uint32_t as = a_mn ? (2048 >> 4) : (32 >> 4), bs = b_mn ? (2048 >> 4) : (32 >> 4);
        uint64_t ad = a0 + off, bd = b0 + off;
        if (!mbar_wait_cluster(bar_tempty + 8 * acc, acc_ph ^ 1, tmo, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * 256;
        uint32_t accum = 0;
        for (int k0 = 0; k0 < kb; k0 += kFfnKps) {
          const int nk = min(kFfnKps, kb - k0);
          if (!mbar_wait(bar_full + 8 * s, ph, tmo, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 2
          for (int i = 0; i < nk; ++i) {
            const uint64_t a = ad + static_cast<uint64_t>(i * (kAStageBytes >> 4));
            const uint64_t b = bd + static_cast<uint64_t>(i * (kAStageBytes >> 4));
            tc_mma_f16_pair(d, a, b, idesc, accum);
            tc_mma_f16_pair(d, a + as, b + bs, idesc, 1u);
            tc_mma_f16_pair(d, a + 2 * as, b + 2 * bs, idesc, 1u);
            tc_mma_f16_pair(d, a + 3 * as, b + 3 * bs, idesc, 1u);
            accum = 1u;
          }
          tc_commit_pair_both(bar_empty + 8 * s);  // free the stage in both CTAs
          if (++s == kFfnStages) {
            s = 0;
            ph ^= 1;
            off = 0;
            ad = a0;
            bd = b0;
          } else {
            off += kFfnStageA >> 4;
            ad += kFfnStageA >> 4;
            bd += kFfnStageB >> 4;
          }
        }
        if (!ok) break;
        tc_commit_pair_both(bar_tfull + 8 * acc);
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1;
      }
      if (!ok) {
        ffn_error(p, 0x41);
        *abort_flag = 1;
      }
      griddep_launch_dependents();
      tc_commit_pair(mapa_shared(bar_drain, 0));
      mbar_wait(bar_drain, 0, kDrainTimeoutNs, nullptr);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - 2, quarter = warp & 3, half = ew >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t buf = sEpi + ew * kEpiBufBytes;
    const uint32_t rowp = buf + lane * 128;
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true, stored = false;
    // Stages 64 columns (32 packed words a lane, its row) and stores them by TMA.
    auto begin = [&]() {
      if (stored) {
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
      }
      stored = true;
    };
    auto put = [&](int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // columns 8 j .. of the 64
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rowp + ((j ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c),
                   "r"(d)
                   : "memory");
    };
    auto end = [&](const CUtensorMap* m, int col, int row, const FfnProblem& q) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row < q.M && col < q.N) {
        tma_store_2d(m, buf, col, row);
        bulk_commit();
      }
    };
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(bar_tempty + 8 * acc, 0));
    };
    for (int u = ffn_next(p, first, cid, ncl); u < p.units && ok; u = ffn_next(p, u + step, cid, ncl)) {
      const FfnUnit un = ffn_unit(p, u);
      const FfnProblem& q = p.prob[un.pr];
      const int row0 = un.tm * kFfnTile + static_cast<int>(rank) * 128 + quarter * 32;
      if (!mbar_wait(bar_tfull + 8 * acc, acc_ph, tmo, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t tb = tmem_base + lane_off + acc * 256;
      if constexpr (EPI == FFN_GATED) {
        const int col = un.tn * 128 + half * 64;
        if (p.save) {
#pragma unroll 1
          for (int w = 0; w < 2; ++w) {  // g, then u, as they are
            begin();
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(tb + w * 128 + half * 64 + sub * 32, r);
              tc_wait_ld_regs(r);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                put(sub * 4 + j, pack2<DT>(__uint_as_float(r[8 * j]), __uint_as_float(r[8 * j + 1])),
                    pack2<DT>(__uint_as_float(r[8 * j + 2]), __uint_as_float(r[8 * j + 3])),
                    pack2<DT>(__uint_as_float(r[8 * j + 4]), __uint_as_float(r[8 * j + 5])),
                    pack2<DT>(__uint_as_float(r[8 * j + 6]), __uint_as_float(r[8 * j + 7])));
            }
            end(&maps.c[1 + w], col, row0, q);
          }
        }
        begin();
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          uint32_t g[32], v[32];
          tmem_ld_32x32b_x32(tb + half * 64 + sub * 32, g);
          tmem_ld_32x32b_x32(tb + 128 + half * 64 + sub * 32, v);
          tc_wait_ld_regs(g);
          tc_pin_regs(v);
          if (sub == 1) release();
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            w[i] = pack2<DT>(gate_act<ACT>(__uint_as_float(g[2 * i])) * __uint_as_float(v[2 * i]),
                             gate_act<ACT>(__uint_as_float(g[2 * i + 1])) * __uint_as_float(v[2 * i + 1]));
#pragma unroll
          for (int j = 0; j < 4; ++j) put(sub * 4 + j, w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
        end(&maps.c[0], col, row0, q);
      } else if constexpr (EPI == FFN_DGATE) {
        const int row = row0 + lane;
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          const int col = un.tn * kFfnTile + half * 128 + ch * 64;
          uint32_t gq[32], uq[32];
          const unsigned short* gp = static_cast<const unsigned short*>(p.g) + row * p.ldg + col;
          const unsigned short* up = static_cast<const unsigned short*>(p.u) + row * p.ldu + col;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            if (row < q.M && col + 8 * j + 8 <= q.N) {
              a = __ldg(reinterpret_cast<const uint4*>(gp) + j);
              b = __ldg(reinterpret_cast<const uint4*>(up) + j);
            } else if (row < q.M && col + 8 * j < q.N) {  // the last, partial eight columns
              uint32_t x[8] = {}, y[8] = {};
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (col + 8 * j + i < q.N) x[i] = gp[8 * j + i], y[i] = up[8 * j + i];
              a = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
              b = make_uint4(y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16);
            }
            gq[4 * j] = a.x, gq[4 * j + 1] = a.y, gq[4 * j + 2] = a.z, gq[4 * j + 3] = a.w;
            uq[4 * j] = b.x, uq[4 * j + 1] = b.y, uq[4 * j + 2] = b.z, uq[4 * j + 3] = b.w;
          }
          begin();
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(tb + half * 128 + ch * 64 + sub * 32, r);
            tc_wait_ld_regs(r);
            if (ch == 1 && sub == 1) release();
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 g2 = unpack2<DT>(gq[sub * 16 + i]), u2 = unpack2<DT>(uq[sub * 16 + i]);
              float dg0, dg1, du0, du1, h0, h1;
              gate_grad<ACT>(__uint_as_float(r[2 * i]), g2.x, u2.x, dg0, du0, h0);
              gate_grad<ACT>(__uint_as_float(r[2 * i + 1]), g2.y, u2.y, dg1, du1, h1);
              w[i] = pack2<DT>(dg0, dg1);
              gq[sub * 16 + i] = pack2<DT>(du0, du1);  // g and u give way to du and h
              uq[sub * 16 + i] = pack2<DT>(h0, h1);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) put(sub * 4 + j, w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          }
          end(&maps.c[0], col, row0, q);
          begin();
#pragma unroll
          for (int j = 0; j < 8; ++j) put(j, gq[4 * j], gq[4 * j + 1], gq[4 * j + 2], gq[4 * j + 3]);
          end(&maps.c[1], col, row0, q);
          begin();
#pragma unroll
          for (int j = 0; j < 8; ++j) put(j, uq[4 * j], uq[4 * j + 1], uq[4 * j + 2], uq[4 * j + 3]);
          end(&maps.c[2], col, row0, q);
        }
      } else {
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          const int col = un.tn * kFfnTile + half * 128 + ch * 64;
          begin();
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(tb + half * 128 + ch * 64 + sub * 32, r);
            tc_wait_ld_regs(r);
            if (ch == 1 && sub == 1) release();
#pragma unroll
            for (int j = 0; j < 4; ++j)
              put(sub * 4 + j, pack2<DT>(__uint_as_float(r[8 * j]), __uint_as_float(r[8 * j + 1])),
                  pack2<DT>(__uint_as_float(r[8 * j + 2]), __uint_as_float(r[8 * j + 3])),
                  pack2<DT>(__uint_as_float(r[8 * j + 4]), __uint_as_float(r[8 * j + 5])),
                  pack2<DT>(__uint_as_float(r[8 * j + 6]), __uint_as_float(r[8 * j + 7])));
          }
          end(&maps.c[un.pr], col, row0, q);
        }
      }
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1;
    }
    if (!ok) {
      ffn_error(p, 0x42);
      *abort_flag = 1;
    }
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still use it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace fo
