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
//              segments with their own operands (dx = dg Wg^T + du Wu^T); a product of few
//              tiles and long K is cut along K into fp32 parts, which the next launch joins
// Operands are K-major or MN-major (read transposed) per problem, so every product of the
// block and its gradients runs on tensors as they are, without a transposition pass.
// h, dg, du (and h again, backward) are rounded to the operands' 16-bit type between the
// products: the matrix instructions take both operands in one type, and a second part, high and
// low, would double these products' work, which is their time.  It costs an output's error
// against 64 bits 0.0017 -> 0.0023 in bf16, 0.00021 -> 0.00029 in fp16 (2-norms of the error over
// that of the result; the output's own rounding is the rest).
//
// Large products are bound by the matrix units under the power limit: 8192 x 4096 x 16384
// bf16, gated 1.5-1.7 ms and down 0.75-0.86 ms (1280-1480 TFLOP/s).  A product of a few waves
// is bound by their number and by what a SM takes from L2 (85 B/ns, which the 256 x 256 tile
// keeps lowest): 1999 x 1024 x 2744 fp16, 27.5 us gated, 17.5 us down and 4.7 us its join;
// backward 1999 x 1024 x 4096, 42 us for dh with its epilogue, 77 us for the gradients.
#pragma once
#include "fo_math.cuh"

namespace fo {

enum : int { FFN_GATED = 0, FFN_DGATE = 1, FFN_GRADS = 2 };
constexpr int kFfnMaxParts = 8;

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
  int parts;           // > 1: units are (tile, part), K blocks [kb part / parts, kb (part + 1) / parts);
                       // part q goes to plane q of an fp32 output
};

struct FfnMaps {
  CUtensorMap a[kFfnMaxProblems][2], b[kFfnMaxProblems][2], c[kFfnMaxProblems];
};

struct FfnParams {
  FfnProblem prob[kFfnMaxProblems];
  int nprob, units, group_m;
  int bf16, save;
  const void *g, *u;  // FFN_DGATE: saved; dg, du and h are written, rows ldo (a multiple of 8) apart
  long long ldg, ldu;
  void *dg, *du, *h;
  long long ldo;
  int* status;
  unsigned long long timeout_ns;
  // Which pair runs a unit: the one that owner[] names (owned), else the pairs take them in turn.
  // Where the first `longs` units are longer and do not come out even (over pairs have one
  // more), the others first take `extra` more of the rest.
  int longs, over, extra;
  int owned;
  unsigned char owner[kFfnOwners];
};

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, uint32_t src, int32_t x, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m), "r"(src), "r"(x),
               "r"(y), "r"(z)
               : "memory");
}

__device__ __forceinline__ void ffn_error(const FfnParams& p, int where) {
  if (atomicCAS(p.status, 0, kStatusTimeout) == 0) {
    p.status[1] = where;
    p.status[2] = static_cast<int>(blockIdx.x);
  }
}

struct FfnUnit {
  int pr, tm, tn, part;
};

__device__ __forceinline__ FfnUnit ffn_unit(const FfnParams& p, int u) {
  FfnUnit r;
  r.pr = 0;
  while (r.pr + 1 < p.nprob && u >= p.prob[r.pr + 1].unit0) ++r.pr;
  const FfnProblem& q = p.prob[r.pr];
  int t = u - q.unit0;
  r.part = 0;
  if (q.parts > 1) {
    const int tiles = q.tiles_m * q.tiles_n;
    r.part = t / tiles;
    t -= r.part * tiles;
  }
  const int per = p.group_m * q.tiles_n;  // rasters of group_m row blocks, for reuse in L2
  const int gr = t / per, in = t - gr * per;
  const int gm = min(p.group_m, q.tiles_m - gr * p.group_m);
  r.tm = gr * p.group_m + in % gm;
  r.tn = in / gm;
  return r;
}

// This pair's next unit after u, and its first one.
__device__ __forceinline__ int ffn_after(const FfnParams& p, int u, int cid, int ncl) {
  if (p.owned) {
    do ++u;
    while (u < p.units && p.owner[u] != cid);
    return u;
  }
  if (p.extra == 0) return u + ncl;
  const int rest = ncl - p.over, mid = p.longs + rest * p.extra;
  if (u < p.longs) return u + ncl < p.longs ? u + ncl : cid >= p.over ? p.longs + cid - p.over : mid + cid;
  if (u < mid) return u + rest < mid ? u + rest : mid + cid;
  return u + ncl;
}
__device__ __forceinline__ int ffn_first(const FfnParams& p, int cid, int ncl) {
  if (p.owned) return ffn_after(p, -1, cid, ncl);
  return p.extra == 0 || cid < p.longs ? cid : p.longs + cid - p.over;
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
    if (EPI != FFN_DGATE) tma_prefetch_desc(&maps.c[0]);
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
      for (int u = ffn_first(p, cid, ncl); u < p.units && ok; u = ffn_after(p, u, cid, ncl)) {
        const FfnUnit un = ffn_unit(p, u);
        const FfnProblem& q = p.prob[un.pr];
        const int arow = un.tm * kFfnTile + static_cast<int>(rank) * 128;
        const int bcol = EPI == FFN_GATED ? un.tn * 128 : un.tn * kFfnTile + static_cast<int>(rank) * 128;
        // everything of the problem in registers: a constant read costs this one thread as
        // much as issuing a copy
        const int a_mn = q.a_mn, b_mn = q.b_mn;
        const int kbeg = q.kb * un.part / q.parts, kb = q.kb * (un.part + 1) / q.parts;
        const int seg = EPI == FFN_GRADS && kbeg >= q.kb0;
        // K blocks left in the segment, the next one's first column
        int left = seg ? q.kb : q.kb0 - kbeg, k = (kbeg - (seg ? q.kb0 : 0)) * kBK;
        const CUtensorMap* ma = &maps.a[un.pr][seg];
        const CUtensorMap* mB = EPI == FFN_GATED ? &maps.b[0][rank] : &maps.b[un.pr][seg];
        for (int k0 = kbeg; k0 < kb; k0 += kFfnKps) {
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
      for (int u = ffn_first(p, cid, ncl); u < p.units && ok; u = ffn_after(p, u, cid, ncl)) {
        const FfnUnit un = ffn_unit(p, u);
        const FfnProblem& q = p.prob[un.pr];
        const int a_mn = q.a_mn, b_mn = q.b_mn;
        const int kbeg = q.kb * un.part / q.parts, kb = q.kb * (un.part + 1) / q.parts;
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
        for (int k0 = kbeg; k0 < kb; k0 += kFfnKps) {
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
    // FFN_DGATE: the two staging blocks in turn: a lane may write one while others still read
    // the other, and meets them at the barrier between.
    int turn = 0;
    auto block = [&]() {
      turn ^= 1;
      return buf + (turn ? 2048u : 0u);
    };
    auto st_block = [&](uint32_t blk, int r, int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(blk + r * 64 + ((j ^ ((r >> 1) & 3)) << 4)), "r"(a), "r"(b),
                   "r"(c), "r"(d)
                   : "memory");
    };
    // 32 rows x 32 columns of g and u: four lanes a row, eight rows a load.
    uint4 pg[EPI == FFN_DGATE ? 4 : 1], pu[EPI == FFN_DGATE ? 4 : 1];
    auto ask_gu = [&](int u, int ch) {
      if constexpr (EPI == FFN_DGATE) {
        const FfnUnit un = ffn_unit(p, u);
        const FfnProblem& q = p.prob[0];
        const int col = un.tn * kFfnTile + half * 128 + ch * 32 + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = un.tm * kFfnTile + static_cast<int>(rank) * 128 + quarter * 32 + i * 8 + (lane >> 2);
          pg[i] = pu[i] = make_uint4(0u, 0u, 0u, 0u);
          const unsigned short* gp = static_cast<const unsigned short*>(p.g) + row * p.ldg + col;
          const unsigned short* up = static_cast<const unsigned short*>(p.u) + row * p.ldu + col;
          if (row < q.M && col + 8 <= q.N) {
            pg[i] = __ldg(reinterpret_cast<const uint4*>(gp));
            pu[i] = __ldg(reinterpret_cast<const uint4*>(up));
          } else if (row < q.M && col < q.N) {  // the last, partial eight columns
            uint32_t x[8] = {}, y[8] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (col + k < q.N) x[k] = gp[k], y[k] = up[k];
            pg[i] = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
            pu[i] = make_uint4(y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16);
          }
        }
      }
    };
    if (EPI == FFN_DGATE) {
      const int u = ffn_first(p, cid, ncl);
      if (u < p.units) ask_gu(u, 0);
    }
    for (int u = ffn_first(p, cid, ncl); u < p.units && ok; u = ffn_after(p, u, cid, ncl)) {
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
            w[i] = pack2<DT>(mul2(gate_act<ACT>(two(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1]))),
                                  two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]))));
#pragma unroll
          for (int j = 0; j < 4; ++j) put(sub * 4 + j, w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
        end(&maps.c[0], col, row0, q);
      } else if constexpr (EPI == FFN_DGATE) {
        // 32 columns at a time.  g and u are asked for one step ahead; they and the results
        // cross HBM as 64 contiguous bytes a row and change hands in shared memory, between
        // that layout and a lane's own row, in two 32 x 64 B blocks a warp.  (TMA stores had
        // to wait for each other's reads of the staging memory: 10 us a tile.)
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          const int col = un.tn * kFfnTile + half * 128 + ch * 32;
          uint32_t gq[16], uq[16];
          auto own_row = [&](const uint4 (&src)[4], uint32_t (&dst)[16]) {
            const uint32_t blk = block();
#pragma unroll
            for (int i = 0; i < 4; ++i) st_block(blk, i * 8 + (lane >> 2), lane & 3, src[i].x, src[i].y, src[i].z, src[i].w);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 v = lds128(blk + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4));
              dst[4 * j] = v.x, dst[4 * j + 1] = v.y, dst[4 * j + 2] = v.z, dst[4 * j + 3] = v.w;
            }
          };
          own_row(pg, gq);
          own_row(pu, uq);
          {  // the next 32 columns, of this tile or of this pair's next one
            int un2 = u;
            if (ch == 3) un2 = ffn_after(p, u, cid, ncl);
            if (un2 < p.units) ask_gu(un2, (ch + 1) & 3);
          }
          uint32_t r[32];
          tmem_ld_32x32b_x32(tb + half * 128 + ch * 32, r);
          tc_wait_ld_regs(r);
          if (ch == 3) release();
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 g2 = unpack2<DT>(gq[i]), u2 = unpack2<DT>(uq[i]);
            Two dg, du, h;
            gate_grad<ACT>(two(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), two(g2.x, g2.y), two(u2.x, u2.y), dg, du, h);
            w[i] = pack2<DT>(dg);
            gq[i] = pack2<DT>(du);  // g and u give way to du and h
            uq[i] = pack2<DT>(h);
          }
          auto store = [&](void* out, const uint32_t (&v)[16]) {
            const uint32_t blk = block();
#pragma unroll
            for (int j = 0; j < 4; ++j) st_block(blk, lane, j, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            __syncwarp();
            const int c = col + (lane & 3) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = i * 8 + (lane >> 2);
              const uint4 t = lds128(blk + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
              unsigned short* dst = static_cast<unsigned short*>(out) + (row0 + rr) * p.ldo + c;
              if (row0 + rr < q.M && c < q.N) *reinterpret_cast<uint4*>(dst) = t;  // rows are padded to 8 columns
            }
          };
          store(p.dg, w);
          store(p.du, gq);
          store(p.h, uq);
        }
      } else if (q.parts > 1) {
        // an fp32 part: 32 columns are a 128-byte row
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          const int col = un.tn * kFfnTile + half * 128 + ch * 32;
          begin();
          uint32_t r[32];
          tmem_ld_32x32b_x32(tb + half * 128 + ch * 32, r);
          tc_wait_ld_regs(r);
          if (ch == 3) release();
#pragma unroll
          for (int j = 0; j < 8; ++j) put(j, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row0 < q.M && col < q.N) tma_store_3d(&maps.c[un.pr], buf, col, row0, un.part);
            bulk_commit();
          }
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

// Joins the fp32 parts [parts][M][ldp] of a product in part order and rounds once.
struct JoinPartsParams {
  const float* part;
  void* out;
  int M, N, parts;
  long long ldp, ldo;
};

template <int DT>
__global__ void __launch_bounds__(256) fo_ffn_join_kernel(const JoinPartsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int per_row = static_cast<int>(p.ldp / 8);  // ldp: N rounded up to 8
  const long long n = static_cast<long long>(p.M) * per_row, plane = p.M * p.ldp;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const int row = static_cast<int>(i / per_row), c = static_cast<int>(i - static_cast<long long>(row) * per_row) * 8;
    const float* src = p.part + row * p.ldp + c;
    float v[8] = {};
#pragma unroll
    for (int q = 0; q < kFfnMaxParts; ++q) {
      if (q >= p.parts) break;
      const float4 a = __ldcg(reinterpret_cast<const float4*>(src + q * plane)), b = __ldcg(reinterpret_cast<const float4*>(src + q * plane) + 1);
      v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    }
    unsigned short* dst = static_cast<unsigned short*>(p.out) + row * p.ldo + c;
    const uint4 w = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
    if (c + 8 <= p.N) {
      *reinterpret_cast<uint4*>(dst) = w;
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.N) dst[j] = static_cast<unsigned short>(u[j / 2] >> (16 * (j & 1)));
    }
  }
}

}  // namespace fo
