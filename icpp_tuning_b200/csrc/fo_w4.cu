// fo_w4.cu -- products of a few tokens with 4-bit weights, out[t, n] = sum_k x[t, k] w[n, k],
// w = scale (q - zero) by groups along k: plain (optional bias) or gated, act(x Wg^T) * (x Wu^T).
//
// Bound by the weights' bytes, and close behind by issue: a SM has to open about 46 weights
// a cycle to keep up with HBM.  So
//   * a warp streams 32 rows (16 and their 16 partners of a gated pair) and its tokens' x in
//     steps of 128 k, by 16-byte cp.async into a ring it keeps for itself, and asks for
//     scales a batch of steps ahead: no block-wide barrier in the loop, and no load whose
//     latency the loop sees;
//   * one ldmatrix hands every lane the 32-bit words (8 weights each) of a 32-k group: of
//     weight row lane / 4, word lane % 4 -- the fragment layout of the m16n8 MMAs when the k
//     order inside a group is that of the words.  The order is free as long as both operands
//     share it.
// A token or a few times large weights (fo_w4i_kernel): the MMA is m16n8k32 on 8-bit integers.
// A word opens into two fragment registers by one shift and two masks, where 16-bit operands
// take three shifts and four masks and half the k an MMA.  x becomes integers first
// (fo_w4_digits_kernel): each token's 128 k's of a step as fixed point of 23 bits, relative to the power of two below
// their largest magnitude, in three 8-bit digits, which are three columns of the MMA.  A
// group's integer sum is exact, and so are 16-bit values within 2^11 of the step's largest; a
// smaller one is off by 2^-22 of that power at most, about what a fp32 sum loses.
// All else (fo_w4_kernel) takes m16n8k16 on 16-bit floats: a word's nibbles pair as (0,4),
// (1,5), (2,6), (3,7), x to match.  A mask and a second constant make each pair the last bits of
// a number whose difference from one of the row's, by its zero, is q - zero, exact: a product is
// x (q - zero) itself, for an infinite x too.  (Opened without the zero, which then left by a
// product with the group's sum(x), a pair took one operation less and a word two MMAs more:
// 4096 x 16384 block, groups of 32 with zeros, 5 tokens fp16 51.0 us against 52.3 now, bf16 57.3
// against 54.8, 32 tokens 149 against 132; and any infinite x gave NaN.)  The digits' zero
// leaves by their sum: both are whole numbers, exact.
// W of a CTA's 8 warps share a tile of rows and split its K (and, for few tiles, the CTAs of a
// cluster): as many as fill the SMs with warps, so that each still walks many steps.  Partial
// sums meet in shared memory (distributed across the cluster) and are added in a fixed order.
//
// Measured, groups of 128 unless said: one token, bf16, 4096 x 16384 gated block (104 MB of
// weights and scales) 30 us with its digits' kernels (16-bit operands: 41); 16384 x 4096
// product 11.3 us; 8 tokens, block 44.2 us; 5 tokens, fp16, groups of 32 with zeros, 52 us (120
// MB).  That last form is bound by the latencies of a step's chain (copies, table, MMAs, sums)
// at 14 warps a SM: its integer pipe is busy 53% of the time, issue 45%.  Short products are
// bound by the launch and the start and end of their few steps a warp (4096 x 4096, one token:
// 5.6 us for 8.7 MB; 5.3 in fp16).  More tokens cost MMAs, 32 of them as much as 4 times
// the bytes: block 64 us at 9 tokens, 122 at 32.
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
  int vec;        // a batch's scales (zeros) of a row are read at once
  int share;      // W: warps that share a tile
  int lg;         // lg of a batch's steps: kBatch or 0
  const void* bias;
  int act;
  void* out;
  long long ldo;
  // The product between the gated block's two kernels travels as two 16-bit parts, high and
  // low, in rows 2 t and 2 t + 1: written so (split), or read so and added (joint; T rows of
  // x, T / 2 of out).
  int split, joint;
  // The digits of x, a record of every step; f32: the output is fp32 (the gated block's inner
  // product).
  const uint8_t* digits;
  int f32;
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

// A word's nibbles as kUnit (q - zero), in 16-bit pairs (0,4), (1,5), (2,6), (3,7).  Exact for
// any zero of 8 bits: all that appears is a whole number of kUnits that the type holds.
template <int DT>
struct W4Open;
template <>
struct W4Open<DT_BF16> {  // the nibble's complement in the last bits of 128: (143 - zero) - (143 - q)
  // in units that keep a step's sum, 128 (q - zero) x, below x: any finite x stays in range
  static constexpr float kUnit = 1.f / 2048;
  uint32_t top;
  __device__ __forceinline__ static uint32_t off(uint32_t zero) {
    const float v = (143.f - static_cast<float>(zero)) * kUnit;
    return pack2<DT_BF16>(v, v);
  }
  __device__ __forceinline__ void set(uint32_t v) { top = v; }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&v)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(v[e]) : "r"(top), "r"(((w >> (4 * e)) & 0x000F000Fu) ^ 0x3D8F3D8Fu));
  }
};
template <>
struct W4Open<DT_F16> {  // a byte's lower nibble in the last bits of 1024, its higher one, as it lies, in those of 64
  static constexpr float kUnit = 1.f;
  uint32_t low, high;    // -(1024 + zero), -(64 + zero)
  __device__ __forceinline__ static uint32_t off(uint32_t zero) { return 0xE400E400u + zero * 0x10001u; }
  __device__ __forceinline__ void set(uint32_t v) {
    low = v;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(high) : "r"(low), "r"(0x63806380u));  // 960
  }
  __device__ __forceinline__ void operator()(uint32_t w, uint32_t (&v)[4]) const {
#pragma unroll
    for (int b = 0; b < 2; ++b, w >>= 8) {
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(v[2 * b]) : "r"((w & 0x000F000Fu) | 0x64006400u), "r"(low));
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(v[2 * b + 1]) : "r"((w & 0x00F000F0u) | 0x54005400u), "r"(high));
    }
  }
};

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

// Which steps a warp takes: batches of 2^lg steps, dealt to the warps in turn, so that a row's
// scales of a whole batch come by one load (a load of every lane's own row costs the SM 32 tag
// lookups whatever its width; 4096 x 16384 block of one token, groups of 64, step by step 47.3
// us, by batches 37.2).  Short K: single steps.
struct W4Steps {
  int first, stride, lg, count;
  __device__ __forceinline__ W4Steps(int warp, int warps, int lg_, int steps) : first(warp), stride(warps), lg(lg_) {
    const int batches = (steps + (1 << lg) - 1) >> lg;
    const int n = first < batches ? (batches - first + stride - 1) / stride : 0;
    // (the last batch may be short)
    count = n == 0 ? 0 : ((n - 1) << lg) + min(1 << lg, steps - ((first + (n - 1) * stride) << lg));
  }
  __device__ __forceinline__ int at(int i) const { return ((first + (i >> lg) * stride) << lg) + (i & ((1 << lg) - 1)); }
};

constexpr int kBatch = 2;  // lg of a batch's steps

// A row's scales and zeros (lane l: row l of the tile): the current batch, the next one under way.
template <int GS, int DT>
struct W4Scales {
  static constexpr int ENT = 4 / GS;  // a step
  const unsigned short* sc;
  const unsigned char* zc;
  int groups;
  static constexpr int kAll = ENT << kBatch, kS = kAll / 4, kZ = kAll > 8 ? 2 : 1;
  uint64_t s[kS], z[kZ], ns[kS], nz[kZ];  // 16-bit scales, 8-bit zeros, the first lowest
  __device__ __forceinline__ void ask(const W4Params& p, int step, int lg) {
#pragma unroll
    for (int i = 0; i < kS; ++i) ns[i] = 0;
#pragma unroll
    for (int i = 0; i < kZ; ++i) nz[i] = 0x0808080808080808ull;
    const int at = step * ENT;  // the entry, where a group is GS blocks
    if (p.vec && lg == kBatch && at + kAll <= groups) {
      if constexpr (kS == 1) {
        ns[0] = __ldg(reinterpret_cast<const unsigned long long*>(sc + at));
        if (zc != nullptr) nz[0] = __ldg(reinterpret_cast<const unsigned*>(zc + at));
      } else {
#pragma unroll
        for (int i = 0; i < kS; i += 2) {
          const ulonglong2 v = __ldg(reinterpret_cast<const ulonglong2*>(sc + at + 4 * i));
          ns[i] = v.x, ns[i + 1] = v.y;
        }
        if (zc != nullptr) {
          if constexpr (kZ == 1) nz[0] = __ldg(reinterpret_cast<const unsigned long long*>(zc + at));
          else {
            const ulonglong2 v = __ldg(reinterpret_cast<const ulonglong2*>(zc + at));
            nz[0] = v.x, nz[1] = v.y;
          }
        }
      }
      return;
    }
    if (GS == 1 && p.vec && lg == 0 && at + 4 <= groups) {
      ns[0] = __ldg(reinterpret_cast<const unsigned long long*>(sc + at));
      if (zc != nullptr) nz[0] = __ldg(reinterpret_cast<const unsigned*>(zc + at));
      return;
    }
    if (GS == 2 && p.vec && lg == 0 && at + 2 <= groups) {
      ns[0] = __ldg(reinterpret_cast<const unsigned*>(sc + at));
      if (zc != nullptr) nz[0] = __ldg(reinterpret_cast<const unsigned short*>(zc + at));
      return;
    }
    if (zc != nullptr)
#pragma unroll
      for (int i = 0; i < kZ; ++i) nz[i] = 0;
#pragma unroll
    for (int e = 0; e < kAll; ++e) {
      if (e >= ENT << lg) break;
      const int i = at + e;
      const int of = GS == 4 ? (p.rcp != 0 ? static_cast<int>(__umulhi(static_cast<uint32_t>(i), p.rcp)) : i)
                     : GS == 2 ? i : i / p.per32;
      const int g = min(of, groups - 1);  // past K: unused
      ns[e / 4] |= static_cast<uint64_t>(__ldg(sc + g)) << (16 * (e & 3));
      if (zc != nullptr) nz[e / 8] |= static_cast<uint64_t>(__ldg(zc + g)) << (8 * (e & 7));
    }
  }
  __device__ __forceinline__ void turn() {
#pragma unroll
    for (int i = 0; i < kS; ++i) s[i] = ns[i];
#pragma unroll
    for (int i = 0; i < kZ; ++i) z[i] = nz[i];
  }
  __device__ __forceinline__ float scale(int e) const {
    return unpack2<DT>(static_cast<uint32_t>(s[0] >> (16 * e)) & 0xFFFFu).x;
  }
  __device__ __forceinline__ uint32_t zero(int e) const { return static_cast<uint32_t>(z[0] >> (8 * e)) & 255u; }
  __device__ __forceinline__ void next() {  // to the next step of the batch
    if constexpr (ENT == 4) {
#pragma unroll
      for (int i = 0; i + 1 < kS; ++i) s[i] = s[i + 1];
    } else if constexpr (kS == 2) {
      s[0] = s[0] >> (16 * ENT) | s[1] << (64 - 16 * ENT), s[1] >>= 16 * ENT;
    } else {
      s[0] >>= 16 * ENT;
    }
    if constexpr (kZ == 2) z[0] = z[0] >> (8 * ENT) | z[1] << (64 - 8 * ENT), z[1] >>= 8 * ENT;
    else z[0] >>= 8 * ENT;
  }
};

// NT: 8-token MMA blocks.
template <int NT>
struct W4Shape {
  static constexpr int kStep = kStepW + 2048 * NT;
  static constexpr int kCtas = NT <= 2 ? 2 : 1;    // a SM
  static constexpr int kTableRow = 48;             // keeps 16-byte stores and 8-byte reads of 8 rows off each other's banks
  static constexpr int kTable = kRows * kTableRow; // a step's (scale, what takes the zero off) pairs, up to 4 a row
  static constexpr int kBudget = (NT <= 2 ? 110 : 200) * 1024 / kWarps - kTable;
  static constexpr int kStages = kBudget / kStep < 6 ? kBudget / kStep : 6;
  static constexpr int kRed = kRows * 8 * NT * 4;  // one warp's sums: its idle ring at the end
  static constexpr int kWarp = ((kStages * kStep > kRed ? kStages * kStep : kRed) + kTable + 127) / 128 * 128;  // bytes of a warp
  static constexpr int kSmem = kWarps * kWarp + kRed;
  static_assert(kStages >= 2, "a ring");
};

// GS: 32-k blocks whose sums share a scale in one step (1, 2 or 4; 1 serves any group size).
// JOINT: x's rows are the two parts of half as many tokens; the ring takes the high ones first,
// and a token's parts meet in one accumulator.
template <bool GATED, int NT, int GS, int DT, bool JOINT>
__global__ void __launch_bounds__(256, W4Shape<NT>::kCtas) fo_w4_kernel(const __grid_constant__ W4Params p) {
  using S = W4Shape<NT>;
  constexpr int NA = JOINT ? NT / 2 : NT;                     // blocks of sums
  constexpr int ENT = 4 / GS, kOut = GATED ? 16 : 32;         // outputs of a tile
  constexpr int kTableRow = S::kTableRow;
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
  const W4Steps turn(rank * W + warp % W, Q * W, p.lg, steps);
  const int mine = n0 < p.N ? turn.count : 0;
  uint8_t* const own = smem_w4 + warp * S::kWarp;
  const uint32_t ring = smem_u32(own);
  uint8_t* const table = own + S::kWarp - S::kTable;

  // Sources of this lane.  Rows past N repeat the last one: nothing of them is stored.  Row
  // block b: the gate's and the up weights' 16 rows, or rows 16 b of the one matrix.
  const char* src[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int m = GATED ? c >> 1 : 0, n = n0 + r + 8 * (GATED ? c & 1 : c);
    src[c] = static_cast<const char*>(p.q[m]) + min(n, p.N - 1) * p.ldq[m] + t * 16;
  }
  const unsigned short* xs = static_cast<const unsigned short*>(p.x) + (tok0 + (JOINT ? 2 : 1) * (lane >> 4)) * p.ldx + (lane & 15) * 8;
  // The four 16-byte blocks of a weight row are stored rotated, odd tokens' halves swapped, so
  // that the reads below fall into distinct banks.
  const uint32_t w_at = (r * 4 + (t ^ ((r >> 1) & 3))) * 16;
  const uint32_t x_at = kStepW + ((lane >> 4) * 16 + ((lane & 15) ^ ((lane >> 4) << 2))) * 16;
  int todo = 0;               // steps asked for
  uint32_t put = ring;        // where the next one goes
  auto issue = [&]() {        // this warp's next step (an empty group past the end)
    if (todo < mine) {
      const int s = turn.at(todo);
      // past K: zeros, and nothing is read
      const uint32_t wn = s * 128 + t * 32 < p.K ? 16u : 0u, xn = s * 128 + (lane & 15) * 8 < p.K ? 16u : 0u;
      const int wo = wn ? s * 64 : 0, xo = xn ? s * 128 : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) cp_async_16(put + w_at + c * 512, src[c] + wo, wn);
#pragma unroll
      for (int c = 0; c < 4 * NT; ++c) {  // two tokens a copy, 16 blocks each
        const int row = !JOINT ? 2 * c : c < 2 * NT ? 4 * c : 4 * c - 8 * NT + 1;  // of its first token
        if (!JOINT && c > 0 && row >= toks) break;
        if (row + (JOINT ? 2 : 1) * (lane >> 4) < toks) cp_async_16(put + x_at + c * 512, xs + row * p.ldx + xo, xn);
      }
    }
    cp_async_commit();
    ++todo;
    put += S::kStep;
    if (put == ring + S::kStages * S::kStep) put = ring;
  };
  // A step's scales and zeros: lane l those of row l.
  const int tm = GATED ? lane >> 4 : 0, tn = min(n0 + (GATED ? lane & 15 : lane), p.N - 1);
  W4Scales<GS, DT> scales;
  scales.sc = static_cast<const unsigned short*>(p.scale[tm]) + tn * p.lds[tm];
  scales.zc = p.zero[tm] == nullptr ? nullptr : p.zero[tm] + tn * p.ldz[tm];
  scales.groups = (p.K + p.per32 * 32 - 1) / (p.per32 * 32);
  const int batch = (1 << p.lg) - 1;

  griddep_wait();
  griddep_launch_dependents();
  if (mine > 0) scales.ask(p, turn.at(0), p.lg);
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) issue();

  float acc[2][NA][4] = {};
  const float none[4] = {0.f, 0.f, 0.f, 0.f};
  // ldmatrix: lane l addresses row l % 8 of row block l / 8
  const uint32_t my_row = (lane >> 3) * 512u + (lane & 7) * 64u, my_rot = ((lane & 7) >> 1) & 3;
  const uint32_t my_x = kStepW + r * 256u, x_rot = (r & 1) << 2;
  uint32_t stage = ring;
  for (int i = 0; i < mine; ++i) {
    __syncwarp();  // the other lanes have read the slot and the table that are refilled next
    const bool fresh_batch = (i & batch) == 0;
    if (fresh_batch) scales.turn();
    uint32_t entry[2 * ENT];
#pragma unroll
    for (int e = 0; e < ENT; ++e) entry[2 * e] = __float_as_uint(scales.scale(e) * (1.f / W4Open<DT>::kUnit)), entry[2 * e + 1] = W4Open<DT>::off(scales.zero(e));
    if constexpr (ENT == 1) {
      *reinterpret_cast<uint2*>(table + lane * kTableRow) = make_uint2(entry[0], entry[1]);
    } else {
#pragma unroll
      for (int e = 0; e < ENT; e += 2)
        *reinterpret_cast<uint4*>(table + lane * kTableRow + e * 8) = make_uint4(entry[2 * e], entry[2 * e + 1], entry[2 * e + 2], entry[2 * e + 3]);
    }
    cp_async_wait<S::kStages - 2>();
    __syncwarp();  // the other lanes' copies and table rows
    issue();
    if (fresh_batch && i + batch + 1 < mine) scales.ask(p, turn.at(i + batch + 1), p.lg);
    scales.next();
    float dot[2][NA][4], by[2][2];  // by: the scales of rows r, r + 8 of both blocks
    W4Open<DT> open[2][2];          // and what takes their zeros off
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t xb[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 d = make_uint4(0u, 0u, 0u, 0u);
        if ((JOINT ? 2 * (nt % NA * 8 + r) : nt * 8 + r) < toks) d = lds128(stage + my_x + nt * 2048 + ((4 * j + t) ^ x_rot) * 16);
        xb[nt][0] = __byte_perm(d.x, d.z, 0x5410u), xb[nt][1] = __byte_perm(d.x, d.z, 0x7632u);
        xb[nt][2] = __byte_perm(d.y, d.w, 0x5410u), xb[nt][3] = __byte_perm(d.y, d.w, 0x7632u);
      }
      uint32_t w[4];
      ldsm4(stage + my_row + ((j ^ my_rot) << 4), w);
      const bool fresh = j % GS == 0;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (fresh) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 v = *reinterpret_cast<const uint2*>(table + (m * 16 + h * 8 + r) * kTableRow + j / GS * 8);
            by[m][h] = __uint_as_float(v.x), open[m][h].set(v.y);
          }
        }
        uint32_t a[2][4];  // {row r, row r + 8} x {pairs 0, 1}, {pairs 2, 3}
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[4];
          open[m][h](w[2 * m + h], v);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e >> 1][(e & 1) * 2 + h] = v[e];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<DT>(dot[m][nt % NA], a[0], xb[nt][0], xb[nt][1], fresh && nt < NA ? none : dot[m][nt % NA]);
          mma_16816<DT>(dot[m][nt % NA], a[1], xb[nt][2], xb[nt][3], dot[m][nt % NA]);
        }
      }
      if ((j + 1) % GS == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int nt = 0; nt < NA; ++nt) {
            const float2 u = both(fma2(two(dot[m][nt][0], dot[m][nt][1]), two(by[m][0]), two(acc[m][nt][0], acc[m][nt][1])));
            const float2 v = both(fma2(two(dot[m][nt][2], dot[m][nt][3]), two(by[m][1]), two(acc[m][nt][2], acc[m][nt][3])));
            acc[m][nt][0] = u.x, acc[m][nt][1] = u.y, acc[m][nt][2] = v.x, acc[m][nt][3] = v.y;
          }
        }
      }
    }
    stage += S::kStep;
    if (stage == ring + S::kStages * S::kStep) stage = ring;
  }

  // Partial sums: the warps of a tile, then the CTAs of the cluster (whose tile is one).
  constexpr int TW = 8 * NA;
  cp_async_wait_all();
  __syncwarp();  // the warp is done with its ring
  float* red = reinterpret_cast<float*>(own);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int nt = 0; nt < NA; ++nt)
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
  const bool fold = !JOINT && p.joint;  // a token's parts are two columns
  const int tokens = p.joint ? (toks + 1) / 2 : toks, each = kOut * tokens;
  for (int o = rank * 256 + threadIdx.x; o < per_cta * each; o += 256 * Q) {
    const int j = o / each, oo = o - j * each;
    const int tok = oo / kOut, f = oo % kOut, col = fold ? 2 * tok : tok;
    const int n = (tile0 + j) * kOut + f, row = (p.joint ? tok0 / 2 : tok0) + tok;
    if (n >= p.N) continue;
    float v = total(j, f * TW + col);
    if (fold) v += total(j, f * TW + col + 1);
    if constexpr (GATED) v = both(gate_act(p.act, two(v))).x * total(j, (16 + f) * TW + col);
    else if (p.bias != nullptr) v += load_vec(p.bias, DT, n);
    const uint32_t hi = pack2<DT>(v, 0.f);
    unsigned short* out = static_cast<unsigned short*>(p.out) + (p.split ? 2 * row : row) * p.ldo + n;
    *out = static_cast<unsigned short>(hi);
    if (p.split) out[p.ldo] = static_cast<unsigned short>(pack2<DT>(low_part(v, unpack2<DT>(hi).x), 0.f));
  }
  if (Q > 1) cluster_sync();  // the others may still read this CTA's sums
}

// ---------------------------------------------------------------------- x as digits
constexpr int kPlanes = 3;

// A step's record: 4 groups x 8 NT columns x 32 digits, then every column's sums over the
// step's ENT blocks, then its scale.  Column 3 t + p is digit p of token t, the first the
// highest; a group's digits are ordered like the fragments: for each word the k of its even
// nibbles, then of its odd ones.  Sums are of the digits, whole numbers.
template <int NT, int GS>
struct W4iShape {
  static constexpr int kEnt = 4 / GS;
  static constexpr int kRec = 1024 * NT + (kEnt + 1) * 32 * NT;
  static constexpr int kStep = kStepW + kRec;
  static constexpr int kTable = kRows * 40;        // a step's (scale, -zero) pairs, up to 4 a row
  static constexpr int kBudget = 113 * 1024 / kWarps - kTable;  // two CTAs a SM
  static constexpr int kStages = kBudget / kStep < 6 ? kBudget / kStep : 6;
  static constexpr int kRed = kRows * 8 * NT * 4;
  static constexpr int kWarp = ((kStages * kStep > kRed ? kStages * kStep : kRed) + kTable) / 16 * 16;
  static constexpr int kSmem = kWarps * kWarp + kRed;
  static_assert(kStages >= 2 && kStep % 16 == 0, "a ring");
};

// x (16-bit or fp32) [T, K] into digit records: sixteen lanes a step of a token.  A step with
// a value that is not finite gets the scale NaN.
struct DigitParams {
  const void* x;
  long long ldx;
  int T, K, steps, dt;
  uint8_t* digits;
};

template <int NT, int GS>
__global__ void __launch_bounds__(256) fo_w4_digits_kernel(const __grid_constant__ DigitParams p) {
  using S = W4iShape<NT, GS>;
  griddep_wait();
  griddep_launch_dependents();
  const int unit = blockIdx.x * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  const int tok = min(unit / p.steps, p.T - 1), step = unit % p.steps, k = step * 128 + l * 8;
  float f[8] = {};
  if (k < p.K) {
    if (p.dt == DT_F32) {
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + tok * p.ldx + k);
      const float4 a = src[0], b = src[1];
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.x) + tok * p.ldx + k);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = p.dt == DT_BF16 ? unpack2<DT_BF16>(w[i]) : unpack2<DT_F16>(w[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
  uint32_t most = 0;  // the largest magnitude's bits: infinities and NaN come out on top
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(fabsf(f[i])));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  const bool fine = most < 0x7F800000u;
  // Units of 2^(e - 21): |v| <= 2^22, which leaves the high digit room for a carry.  A power of
  // two, so that a 16-bit value within 2^11 of the largest is exact.  (Its inverse by two
  // factors: one would leave the range for small values.)
  const int e = max(static_cast<int>(most >> 23), 1) - 127, up = 21 - e, up1 = up / 2, up2 = up - up1;
  const float s1 = __int_as_float((up1 + 127) << 23), s2 = __int_as_float((up2 + 127) << 23);
  int d[kPlanes][8], sum[kPlanes] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int v = fine ? __float2int_rn(f[i] * s1 * s2) : 0;
    d[2][i] = static_cast<int8_t>(v);
    const int v1 = (v - d[2][i]) >> 8;
    d[1][i] = static_cast<int8_t>(v1);
    d[0][i] = (v1 - d[1][i]) >> 8;
#pragma unroll
    for (int q = 0; q < kPlanes; ++q) sum[q] += d[q][i];
  }
#pragma unroll
  for (int q = 0; q < kPlanes; ++q)
#pragma unroll
    for (int o = 1; o < 4 * GS; o <<= 1) sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], o);  // a block's 4 GS words
  if (unit >= p.T * p.steps) return;
  uint8_t* rec = p.digits + static_cast<long long>(step) * S::kRec;
#pragma unroll
  for (int q = 0; q < kPlanes; ++q) {
    uint2 w = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w.x |= (d[q][2 * i] & 255u) << (8 * i);
      w.y |= (d[q][2 * i + 1] & 255u) << (8 * i);
    }
    const int col = tok * kPlanes + q;
    *reinterpret_cast<uint2*>(rec + (l >> 2) * (256 * NT) + col * 32 + (l & 3) * 8) = w;
    float* tail = reinterpret_cast<float*>(rec + 1024 * NT) + col;
    // the digit's unit; it may be subnormal, and its integers still scale exactly
    const float unit_q = fine ? ldexpf(1.f, 8 * (kPlanes - 1 - q) - up) : __int_as_float(0x7FC00000);
    if ((l & (4 * GS - 1)) == 0) tail[l / (4 * GS) * (8 * NT)] = static_cast<float>(sum[q]);
    if (l == 0) tail[S::kEnt * 8 * NT] = unit_q;
  }
}

__device__ __forceinline__ void imma_16832(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int* c) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

template <bool GATED, int NT, int GS, int DT>
__global__ void __launch_bounds__(256, 2) fo_w4i_kernel(const __grid_constant__ W4Params p) {
  using S = W4iShape<NT, GS>;
  constexpr int ENT = S::kEnt, kOut = GATED ? 16 : 32;
  extern __shared__ __align__(128) uint8_t smem_w4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  int rank, Q;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(Q));
  const int W = p.share, per_cta = kWarps / W;
  const int tile0 = static_cast<int>(blockIdx.x / Q) * per_cta;
  const int n0 = (tile0 + warp / W) * kOut;
  const int cols = kPlanes * p.T;
  const int steps = (p.K + 127) / 128;
  const W4Steps turn(rank * W + warp % W, Q * W, p.lg, steps);
  const int mine = n0 < p.N ? turn.count : 0;
  uint8_t* const own = smem_w4 + warp * S::kWarp;
  const uint32_t ring = smem_u32(own);
  uint8_t* const table = own + S::kWarp - S::kTable;

  const char* src[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int m = GATED ? c >> 1 : 0, n = n0 + r + 8 * (GATED ? c & 1 : c);
    src[c] = static_cast<const char*>(p.q[m]) + min(n, p.N - 1) * p.ldq[m] + t * 16;
  }
  const uint32_t w_at = (r * 4 + (t ^ ((r >> 1) & 3))) * 16;
  int todo = 0, xtodo = 0;
  auto weights = [&](int i) {  // step i's weights
    if (i < mine) {
      const int s = turn.at(i);
      const uint32_t put = ring + i % S::kStages * S::kStep, wn = s * 128 + t * 32 < p.K ? 16u : 0u;
      const int wo = wn ? s * 64 : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) cp_async_16(put + w_at + c * 512, src[c] + wo, wn);
    }
  };
  auto digits = [&](int i) {  // and its digits (used columns only) and their sums
    if (i < mine) {
      const uint32_t put = ring + i % S::kStages * S::kStep + kStepW;
      const uint8_t* rec = p.digits + static_cast<long long>(turn.at(i)) * S::kRec;
#pragma unroll
      for (int c = 0; c < 2 * NT; ++c) {
        const int at = c * 32 + lane;  // 16-byte block: group, column, half
        if (at / 2 % (8 * NT) < cols) cp_async_16(put + at * 16, rec + at * 16, 16u);
      }
      if (lane < (ENT + 1) * 2 * NT) cp_async_16(put + 1024 * NT + lane * 16, rec + 1024 * NT + lane * 16, 16u);
    }
    cp_async_commit();
  };
  const int tm = GATED ? lane >> 4 : 0, tn = min(n0 + (GATED ? lane & 15 : lane), p.N - 1);
  W4Scales<GS, DT> scales;
  scales.sc = static_cast<const unsigned short*>(p.scale[tm]) + tn * p.lds[tm];
  scales.zc = p.zero[tm] == nullptr ? nullptr : p.zero[tm] + tn * p.ldz[tm];
  scales.groups = (p.K + p.per32 * 32 - 1) / (p.per32 * 32);
  const int batch = (1 << p.lg) - 1;

  // The weights and scales are final before the digits' kernel ends (it began after whatever
  // wrote them), the digits are not.
  if (mine > 0) scales.ask(p, turn.at(0), p.lg);
#pragma unroll
  for (; todo < S::kStages - 1; ++todo) weights(todo);
  for (int i = lane; i < S::kStages * (S::kRec / 16); i += 32) {  // columns without a digit stay zero
    const int st = i / (S::kRec / 16), b = i - st * (S::kRec / 16);
    if (b < 64 * NT && b / 2 % (8 * NT) >= cols) *reinterpret_cast<uint4*>(own + st * S::kStep + kStepW + b * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  griddep_wait();
  griddep_launch_dependents();
#pragma unroll
  for (; xtodo < S::kStages - 1; ++xtodo) digits(xtodo);

  float acc[2][NT][4] = {};
  const int none[4] = {0x4B400000, 0x4B400000, 0x4B400000, 0x4B400000};  // 1.5 * 2^23: an integer added to its bits
  const Two none2 = two(-12582912.f);                                    // is added to its value
  const uint32_t my_row = (lane >> 3) * 512u + (lane & 7) * 64u, my_rot = ((lane & 7) >> 1) & 3;
  const uint32_t my_x = kStepW + lane * 8u;
  int slot = 0;
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();  // other lanes' copies, and their reads of the slot and the table refilled next
    const bool fresh_batch = (i & batch) == 0;
    if (fresh_batch) scales.turn();
#pragma unroll
    for (int e = 0; e < ENT; ++e) {
      const float v = scales.scale(e), z = static_cast<float>(scales.zero(e));
      *reinterpret_cast<float2*>(table + lane * 40 + e * 8) = make_float2(v, -z);
    }
    __syncwarp();
    weights(i + S::kStages - 1);
    digits(i + S::kStages - 1);
    if (fresh_batch && i + batch + 1 < mine) scales.ask(p, turn.at(i + batch + 1), p.lg);
    scales.next();
    const uint32_t stage = ring + slot * S::kStep;
    const uint8_t* stage_p = own + slot * S::kStep;
    int dot[2][NT][4];
    Two unit[NT];  // of this lane's two columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 v = *reinterpret_cast<const float2*>(stage_p + kStepW + 1024 * NT + ENT * (32 * NT) + (nt * 8 + 2 * t) * 4);
      unit[nt] = two(v.x, v.y);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(b[nt][0]), "=r"(b[nt][1]) : "r"(stage + my_x + j * (256 * NT) + nt * 256) : "memory");
      uint32_t w[4];
      ldsm4(stage + my_row + ((j ^ my_rot) << 4), w);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint32_t a[4];  // rows r, r + 8 of the even nibbles, then of the odd ones
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          a[h] = w[2 * m + h] & 0x0F0F0F0Fu;
          a[2 + h] = (w[2 * m + h] >> 4) & 0x0F0F0F0Fu;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) imma_16832(dot[m][nt], a, b[nt][0], b[nt][1], j % GS == 0 ? none : dot[m][nt]);
      }
      if ((j + 1) % GS == 0) {
        Two sx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 v = *reinterpret_cast<const float2*>(stage_p + kStepW + 1024 * NT + j / GS * (32 * NT) + (nt * 8 + 2 * t) * 4);
          sx[nt] = two(v.x, v.y);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float2 lo = *reinterpret_cast<const float2*>(table + (m * 16 + r) * 40 + j / GS * 8);
          const float2 hi = *reinterpret_cast<const float2*>(table + (m * 16 + r + 8) * 40 + j / GS * 8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const Two d01 = add2(two(__int_as_float(dot[m][nt][0]), __int_as_float(dot[m][nt][1])), none2);
            const Two d23 = add2(two(__int_as_float(dot[m][nt][2]), __int_as_float(dot[m][nt][3])), none2);
            // sums of (q - zero) digit: whole numbers below 2^23, exact
            const float2 u = both(fma2(fma2(sx[nt], two(lo.y), d01), mul2(two(lo.x), unit[nt]), two(acc[m][nt][0], acc[m][nt][1])));
            const float2 v = both(fma2(fma2(sx[nt], two(hi.y), d23), mul2(two(hi.x), unit[nt]), two(acc[m][nt][2], acc[m][nt][3])));
            acc[m][nt][0] = u.x, acc[m][nt][1] = u.y, acc[m][nt][2] = v.x, acc[m][nt][3] = v.y;
          }
        }
      }
    }
    if (++slot == S::kStages) slot = 0;
  }

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
  auto total = [&](int j, int row, int tok) {  // a token's digits joined, lowest first
    float v = 0.f;
#pragma unroll
    for (int q = kPlanes - 1; q >= 0; --q) {
      const int i = row * TW + tok * kPlanes + q;
      float d = 0.f;
      if (Q == 1) d = of_tile(j, i);
      else
        for (int c = 0; c < Q; ++c) d += ld_cluster_f32(mapa_shared(pa + i * 4, c));
      v += d;
    }
    return v;
  };
  for (int o = rank * 256 + threadIdx.x; o < per_cta * kOut * p.T; o += 256 * Q) {
    const int j = o / (kOut * p.T), oo = o - j * (kOut * p.T);
    const int tok = oo / kOut, f = oo % kOut, n = (tile0 + j) * kOut + f;
    if (n >= p.N) continue;
    float v = total(j, f, tok);
    if constexpr (GATED) v = both(gate_act(p.act, two(v))).x * total(j, 16 + f, tok);
    else if (p.bias != nullptr) v += load_vec(p.bias, DT, n);
    if (p.f32) static_cast<float*>(p.out)[tok * p.ldo + n] = v;
    else static_cast<unsigned short*>(p.out)[tok * p.ldo + n] = static_cast<unsigned short>(pack2<DT>(v, 0.f));
  }
  if (Q > 1) cluster_sync();  // the others may still read this CTA's sums
}

// ---------------------------------------------------------------------- host
// Tiles, warps a tile and CTAs a tile: as many warps as fit at once (a fifth more is better
// than half as many), then CTAs for a tile of long K, or where most SMs would have none.  Of one
// token 4096 x 4096: 8 warps 5.1 us, 16 in two CTAs 6.5; 16384 x 4096: 4 warps a tile 10.8, 8
// (two waves) 13.0; 64 tokens 4096 x 4096: 8 warps 23.6 (22.2 since the weights open as q -
// zero), 16 29.4.
struct W4Plan {
  int share, q, lg;
  unsigned ctas;
};

W4Plan w4_plan(int N, int K, int out, int chunks, int ctas_a_sm, int batch, int sms) {
  const long long tiles = (N + out - 1) / out, fit = 6ll * kWarps * ctas_a_sm * sms / 5;
  const int steps = (K + 127) / 128;
  int W = 1, Q = 1;
  while (W < kWarps && 2 * tiles * chunks * W <= fit && steps >= 2 * W) W *= 2;
  auto ctas = [&] { return tiles * chunks * Q; };
  while (W == kWarps && Q < 8 && 2 * ctas() <= ctas_a_sm * sms &&
         (steps >= 16 * kWarps * Q || (2 * ctas() <= sms && steps >= 2 * kWarps * Q)))
    Q *= 2;
  // batches only where every warp has whole ones
  return {W, Q, steps >> batch >= W * Q ? batch : 0, static_cast<unsigned>((tiles + kWarps / W - 1) / (kWarps / W) * Q)};
}

template <bool GATED, int NT, int GS, int DT, bool JOINT = false>
cudaError_t launch(W4Params p, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0};
  const int chunks = (p.T + 8 * NT - 1) / (8 * NT);
  const W4Plan l = w4_plan(p.N, p.K, GATED ? 16 : 32, chunks, W4Shape<NT>::kCtas, kBatch, sms);
  p.share = l.share, p.lg = l.lg;
  return launch_pdl(fo_w4_kernel<GATED, NT, GS, DT, JOINT>, opted, dim3(l.ctas, chunks), dim3(256), W4Shape<NT>::kSmem, l.q, stream, p);
}

int64_t digit_blocks(int64_t T) { return (kPlanes * T + 7) / 8; }
// Whether x travels as digits: where the tokens' digits fill one block of 8 columns (4096 x
// 16384 block, bf16, one token: groups of 128 41.1 -> 29.8 us, of 64 43.5 -> 31.8, of 32 48.7 ->
// 39.3); up to three where a group is a step or longer (4 tokens 43.2 -> 33.2, 8 tokens 48.5 ->
// 43.9; groups of 32, 3 tokens: 49.8 -> 54.5).  Up to 2^24 weights a block the second launch
// costs the caller more (3 us) than the GPU saves (one token 4096 x 4096 5.6 -> 6.1, 8192 x 4096
// 8.7 -> 8.2, 16384 x 4096 14.3 -> 11.2; 4 tokens 8192 x 4096 9.1 -> 9.9; 8 tokens 16384 x 4096
// 15.9 -> 16.4).
bool as_digits(int64_t T, int64_t N, int64_t K, int per32) {
  return T > 0 && digit_blocks(T) <= (per32 % 4 == 0 ? 3 : 1) && N * K > digit_blocks(T) << 24;
}
// Bytes of the digit records.
size_t digit_bytes(int64_t T, int64_t K, int per32) {
  const int ent = per32 % 4 == 0 ? 1 : per32 == 2 ? 2 : 4;
  return static_cast<size_t>((K + 127) / 128 * digit_blocks(T) * (1024 + (ent + 1) * 32));
}

// x_dt: of p.x.  `room` holds digit_bytes.
template <bool GATED, int NT, int GS, int DT>
cudaError_t launch_digits(W4Params p, int x_dt, void* room, int sms, cudaStream_t stream) {
  static std::atomic<uint64_t> opted{0}, none{0};
  DigitParams d = {};
  d.x = p.x, d.ldx = p.ldx, d.T = p.T, d.K = p.K, d.steps = (p.K + 127) / 128, d.dt = x_dt;
  d.digits = static_cast<uint8_t*>(room);
  const unsigned blocks = static_cast<unsigned>((d.T * d.steps + 15) / 16);
  cudaError_t e = launch_pdl(fo_w4_digits_kernel<NT, GS>, none, dim3(blocks), dim3(256), 0, 1, stream, d);
  if (e != cudaSuccess) return e;
  const W4Plan l = w4_plan(p.N, p.K, GATED ? 16 : 32, 1, 2, kBatch, sms);
  p.share = l.share, p.lg = l.lg, p.digits = d.digits;
  return launch_pdl(fo_w4i_kernel<GATED, NT, GS, DT>, opted, dim3(l.ctas), dim3(256), W4iShape<NT, GS>::kSmem, l.q, stream, p);
}

template <bool GATED, int GS, int DT>
cudaError_t by_tokens(const W4Params& p, int x_dt, void* room, int sms, cudaStream_t s) {
  if (room != nullptr) {
    if constexpr (GS == 4) {
      if (digit_blocks(p.T) == 3) return launch_digits<GATED, 3, GS, DT>(p, x_dt, room, sms, s);
      if (digit_blocks(p.T) == 2) return launch_digits<GATED, 2, GS, DT>(p, x_dt, room, sms, s);
    }
    return launch_digits<GATED, 1, GS, DT>(p, x_dt, room, sms, s);
  }
  if (p.T <= 8) return launch<GATED, 1, GS, DT>(p, sms, s);
  if constexpr (!GATED) {
    if (p.joint) return p.T <= 16 ? launch<GATED, 2, GS, DT, true>(p, sms, s) : launch<GATED, 4, GS, DT, true>(p, sms, s);
  }
  if (p.T <= 16) return launch<GATED, 2, GS, DT>(p, sms, s);
  return launch<GATED, 4, GS, DT>(p, sms, s);
}

template <bool GATED, int DT>
cudaError_t by_group(const W4Params& p, int x_dt, void* room, int sms, cudaStream_t s) {
  if (p.per32 % 4 == 0) return by_tokens<GATED, 4, DT>(p, x_dt, room, sms, s);
  if (p.per32 == 2) return by_tokens<GATED, 2, DT>(p, x_dt, room, sms, s);
  return by_tokens<GATED, 1, DT>(p, x_dt, room, sms, s);
}

int check_weight(const FoW4* w, int64_t K, const char* name) {
  if (w->q == nullptr || w->scales == nullptr || !host_aligned16(w->q))
    return host_fail(FO_EINVAL, "%s: q and scales must be device pointers, q 16-byte aligned", name);
  if (w->group <= 0 || w->group % 32 != 0) return host_fail(FO_EINVAL, "%s: group must be a positive multiple of 32, got %d", name, w->group);
  // a step's group comes from a 32-bit reciprocal, exact while steps * steps a group <= 2^32
  if (w->group < K && K / 128 * (w->group / 128) > (1ll << 32))
    return host_fail(FO_EUNSUPPORTED, "%s: K = %lld in groups of %d exceeds K * group = 2^46", name, static_cast<long long>(K), w->group);
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

// room: for the digits of x, of type x_dt; null: x as it is.
int run(W4Params p, bool gated, int dtype, int x_dt, void* room, const HostDevice& hd, cudaStream_t st) {
  const uint32_t per = static_cast<uint32_t>(p.per32) / 4;  // steps a group
  p.rcp = per > 1 ? static_cast<uint32_t>((0x100000000ull + per - 1) / per) : 0u;
  // a batch's scales and zeros of a row: `all` entries, loads of up to 16 bytes
  p.vec = p.per32 == 1 || p.per32 == 2 || p.per32 == 4;
  const int all = p.vec ? 16 / p.per32 : 1, part = all < 8 ? all : 8;
  for (int m = 0; m < (gated ? 2 : 1); ++m)
    p.vec = p.vec && p.lds[m] % part == 0 && reinterpret_cast<uintptr_t>(p.scale[m]) % (2 * part) == 0 &&
            (p.zero[m] == nullptr || (p.ldz[m] % all == 0 && reinterpret_cast<uintptr_t>(p.zero[m]) % all == 0));
  const bool bf = dtype == FO_DT_BF16;
  const cudaError_t e = gated ? (bf ? by_group<true, DT_BF16>(p, x_dt, room, hd.sms, st) : by_group<true, DT_F16>(p, x_dt, room, hd.sms, st))
                              : (bf ? by_group<false, DT_BF16>(p, x_dt, room, hd.sms, st) : by_group<false, DT_F16>(p, x_dt, room, hd.sms, st));
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(room != nullptr ? 2 : 1);
  return FO_OK;
}

}  // namespace
}  // namespace fo

extern "C" size_t fo_matvec_w4_workspace_size(const FoMatvecW4Desc* d) {
  if (d == nullptr || d->K <= 0 || d->w.group < 32) return 0;
  return fo::as_digits(d->T, d->N, d->K, d->w.group / 32) ? fo::digit_bytes(d->T, d->K, d->w.group / 32) : 0;
}

extern "C" int fo_matvec_w4(const FoMatvecW4Desc* d, void* stream) {
  using namespace fo;
  if (d == nullptr) return host_fail(FO_EINVAL, "null descriptor");
  if (int rc = check_sizes(d->T, d->N, d->K, d->dtype)) return rc;
  if (d->T == 0 || d->N == 0) return host_ok();
  if (d->K == 0) return host_fail(FO_EINVAL, "K must be positive");
  if (int rc = check_weight(&d->w, d->K, "w")) return rc;
  if (int rc = check_x(d->x, d->ldx, d->T, d->K)) return rc;
  if (d->out == nullptr || d->ldo < d->N) return host_fail(FO_EINVAL, "out must be a device pointer with rows of N values or more");
  const size_t need = fo_matvec_w4_workspace_size(d);
  if (need > 0 && (d->workspace == nullptr || d->workspace_bytes < need || !host_aligned16(d->workspace)))
    return host_fail(FO_EINVAL, "needs a 16-byte aligned workspace of %zu bytes", need);
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  W4Params p = {};
  p.x = d->x, p.ldx = d->ldx, p.T = static_cast<int>(d->T), p.N = static_cast<int>(d->N), p.K = static_cast<int>(d->K);
  set_weight(&p, 0, &d->w);
  p.per32 = d->w.group / 32;
  p.bias = d->bias, p.out = d->out, p.ldo = d->ldo;
  if (int rc = run(p, false, d->dtype, d->dtype == FO_DT_BF16 ? DT_BF16 : DT_F16, need > 0 ? d->workspace : nullptr, hd,
                   static_cast<cudaStream_t>(stream)))
    return rc;
  return host_ok();
}

namespace fo {
namespace {

// The gated block's workspace: the product between, in fp32 to become digits, else in two
// 16-bit parts (either way 4 bytes a value); then the digits, x's and later the product's.
struct GatedW4Plan {
  bool digits;  // of x and of the product between
  size_t h, room;
  explicit GatedW4Plan(const FoGatedFfnW4Desc* d) {
    const int g1 = d->w_gate.group / 32, g2 = d->w_down.group / 32;
    digits = as_digits(d->T, 2 * d->F, d->D, g1) && as_digits(d->T, d->N, d->F, g2);
    h = (static_cast<size_t>(d->T) * ((d->F + 7) / 8 * 8) * 4 + 255) / 256 * 256;
    const size_t a = digit_bytes(d->T, d->D, g1), b = digit_bytes(d->T, d->F, g2);
    room = digits ? (a > b ? a : b) : 0;
  }
};

}  // namespace
}  // namespace fo

extern "C" size_t fo_gated_ffn_w4_workspace_size(const FoGatedFfnW4Desc* d) {
  if (d == nullptr || d->T <= 0 || d->D <= 0 || d->F <= 0 || d->w_gate.group < 32 || d->w_down.group < 32) return 0;
  const fo::GatedW4Plan plan(d);
  return plan.h + plan.room;
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
  const int dt = d->dtype == FO_DT_BF16 ? DT_BF16 : DT_F16;
  const GatedW4Plan plan(d);
  char* const room = static_cast<char*>(d->workspace) + plan.h;
  p.f32 = plan.digits, p.split = !plan.digits;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = run(p, true, d->dtype, dt, plan.digits ? room : nullptr, hd, st)) return rc;
  W4Params o = {};
  o.x = d->workspace, o.ldx = p.ldo, o.T = plan.digits ? p.T : 2 * p.T, o.N = static_cast<int>(d->N), o.K = p.N;
  set_weight(&o, 0, &d->w_down);
  o.per32 = d->w_down.group / 32;
  o.out = d->out, o.ldo = d->ldo;
  o.joint = !plan.digits;
  if (int rc = run(o, false, d->dtype, plan.digits ? DT_F32 : dt, plan.digits ? room : nullptr, hd, st)) return rc;
  return host_ok();
}
