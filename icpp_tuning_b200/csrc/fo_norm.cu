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
// W warps own a row, 8 or 16 columns a thread; the CTAs walk the rows side by side.
// Rows arrive by bulk copies in a ring of shared memory, several rows ahead, so the copies
// never wait for a row's reductions.  A row that does not start or end on a 16-byte boundary
// is copied as the 16-byte blocks around it, as far as they lie inside its tensor; what is
// left of the tensor's first and last block is read directly.  Each value crosses HBM once:
// both kernels are bound by HBM.
// Statistics are fp32, of centred values in the LayerNorm form.  The backward pass needs one
// round of sums a row (two in the LayerNorm form): mean(e yhat) is linear in t, so its three
// parts sum(A y dr), sum(A y c), sum(A y r), A = gate w_post, join the round that gives rho
// and mean(c rhat).  Of the parameter gradients only sum(dz rhat), q = sum(t yhat) (and
// sum(dz), sum(t) with biases) are carried: dw_post = gate q, dgate = w_post q + b_post
// sum(t), db_post = gate sum(t) are formed once a gate row, in the kernel that joins the
// CTAs' sums in a fixed order.
//
// Measured, 16384 x 4096 bf16 with gate: RMS forward 91 us (5.9 TB/s), backward 142 us (5.7
// TB/s); LayerNorm 114 and 243.  Odd rows cost instructions, one 2-byte shared load and store a
// value: LayerNorm backward 4680 x 1001 fp16, 42 us (1000 columns: 28).  The LayerNorm-form and
// odd-row kernels are bound by instructions at 16 warps a SM, and their backward passes spill at
// the cap of 128 registers: 72 to 104 bytes a thread in the LayerNorm form up to 4096 columns
// (716 above), 104 to 152 (364) for odd rms rows, 180 to 320 (864) for odd LayerNorm rows; the
// other rms ones 64 at most.  Forward, odd rows of up to 4096 columns spill 150 to 172, all rows
// of more than 8192 columns 120 to 690.
#include "fo_host.cuh"
#include "fo_math.cuh"
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
  // work units: `chunks` to a gate group, its rows in turn; backward, the sums of unit u go to
  // part[u][k][ldp] (k: dz rhat, t yhat; in the LayerNorm form dz, t)
  int groups, chunks;
  int ldp;
  float* part;
  int* status;
  unsigned long long timeout_ns;
};

// Where a thread's NP pairs of columns lie.  VEC 8: pair e is columns 2 (e % 4) of the
// 16-byte block (e / 4) * 32 W + tid; VEC 1: the single columns 2 e * 32 W + tid and
// (2 e + 1) * 32 W + tid.
template <int W, int VEC>
struct Cols {
  int tid, D;
  __device__ __forceinline__ int first(int e) const { return VEC == 8 ? ((e >> 2) * 32 * W + tid) * 8 + 2 * (e & 3) : 2 * e * 32 * W + tid; }
  __device__ __forceinline__ int second(int e) const { return VEC == 8 ? first(e) + 1 : first(e) + 32 * W; }
  __device__ __forceinline__ bool in(int e) const { return first(e) < D; }        // VEC 8: both columns
  __device__ __forceinline__ bool in2(int e) const { return VEC == 8 ? in(e) : second(e) < D; }
  // VEC 1: a thread's i-th column (of 2 NP) can lie past the row: layouts take more than half
  // of their columns, but for the smallest.
  __device__ __forceinline__ static constexpr bool maybe_out(int i, int np) { return i >= np || (W == 1 && np == 4); }
};

// A parameter vector's pairs; `fill` where it is absent, 0 past D.  Every load is in bounds
// and unconditional, so that they are all under way at once.
template <int W, int VEC, int NP>
__device__ __forceinline__ void load_param(const void* ptr, int dt, const Cols<W, VEC>& c, float fill, Two (&f)[NP]) {
  float v[2 * NP];
  if (ptr == nullptr) {
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) v[i] = fill;
  } else if constexpr (VEC == 8) {
#pragma unroll
    for (int e = 0; e < NP; e += 4) {
      float t[8];
      load_vec8(ptr, dt, min(c.first(e), c.D - 8), t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[2 * e + i] = t[i];
    }
  } else if (dt == DT_F32) {
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) v[i] = __ldg(static_cast<const float*>(ptr) + min(c.tid + i * 32 * W, c.D - 1));
  } else {
    unsigned short raw[2 * NP];
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) raw[i] = __ldg(static_cast<const unsigned short*>(ptr) + min(c.tid + i * 32 * W, c.D - 1));
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) v[i] = dt == DT_BF16 ? __bfloat162float(__ushort_as_bfloat16(raw[i])) : __half2float(__ushort_as_half(raw[i]));
  }
#pragma unroll
  for (int e = 0; e < NP; ++e) f[e] = two(c.in(e) ? v[2 * e] : 0.f, c.in2(e) ? v[2 * e + 1] : 0.f);
}

// Pairs e0 .. e0 + 3.
template <int DT, int W, int VEC>
__device__ __forceinline__ void store_row(void* row, const Cols<W, VEC>& c, int e0, const Two (&f)[4]) {
  unsigned short* p = static_cast<unsigned short*>(row);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = both(f[i]);
    w[i] = pack2<DT>(v.x, v.y);
  }
  if constexpr (VEC == 8) {
    if (c.in(e0)) *reinterpret_cast<uint4*>(p + c.first(e0)) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c.in(e0 + i)) p[c.first(e0 + i)] = static_cast<unsigned short>(w[i] & 0xFFFFu);
      if (c.in2(e0 + i)) p[c.second(e0 + i)] = static_cast<unsigned short>(w[i] >> 16);
    }
  }
}

__device__ __forceinline__ const void* vec_at(const void* ptr, int dt, long long i) {
  return ptr == nullptr ? nullptr : static_cast<const char*>(ptr) + i * (dt == DT_F32 ? 4 : 2);
}

// Sums of N <= 16 values over a warp: each butterfly step halves the values a lane carries
// (value i ends in the lanes with those bits), so 8 values take 9 shuffles instead of 40.
template <int N>
__device__ __forceinline__ float warp_sums(const float (&v)[N], int lane) {
  constexpr int M = N <= 8 ? 8 : 16;
  float a[M];
#pragma unroll
  for (int i = 0; i < M; ++i) a[i] = i < N ? v[i] : 0.f;
#pragma unroll
  for (int o = M / 2; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      if (i >= N) continue;  // both halves empty
      const float keep = up ? a[i + o] : a[i], give = up ? a[i] : a[i + o];
      a[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (int o = M; o < 32; o <<= 1) a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
  return a[0];  // lane l: the warp's sum of value l & (M - 1)
}

// Sums over the W warps of a row.  Rounds alternate between two halves of the scratch: a
// warp enters round k + 2 only after every warp has read round k (the barrier of round
// k + 1 lies between), so one barrier a round is enough.
template <int W>
struct RowSum {
  float* red;  // [2][W][16] of this row group
  int round, bar;
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    const int lane = threadIdx.x & 31;
    if constexpr (N == 1) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      if constexpr (W > 1) {
        float* s = red + round * 16 * W;
        if (lane == 0) s[threadIdx.x >> 5] = v[0];
        named_bar_sync(bar, 32 * W);
        v[0] = s[lane & (W - 1)];
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        round ^= 1;
      }
      return;
    }
    constexpr int M = N <= 8 ? 8 : 16, kPer = 32 / M;  // warps whose sums the lanes read at once
    float mine = warp_sums(v, lane);                   // lane l: value l & (M - 1)
    if constexpr (W > 1) {
      float* s = red + round * 16 * W;
      if (lane < M) s[(threadIdx.x >> 5) * M + lane] = mine;
      named_bar_sync(bar, 32 * W);
      mine = 0.f;
#pragma unroll
      for (int w = 0; w < W; w += kPer)
        if (W >= kPer || lane / M < W) mine += s[w * M + lane];
#pragma unroll
      for (int o = M; o < 32; o <<= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      round ^= 1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, mine, i);
  }
};

constexpr int kCtaWarps = 8;
constexpr int row_groups(int W) { return W >= kCtaWarps ? 1 : kCtaWarps / W; }
constexpr int kBwdStages = 3;

// Bytes of one row in the ring: every column a row group's threads hold (those past the row
// stay zero), and with VEC 1 up to a 16-byte block more on either side.
template <int W, int NP, int VEC>
constexpr int ring_row() {
  return NP * 2 * 32 * W * 2 + (VEC == 8 ? 0 : 32);
}

// One row group's ring and its columns: NT rows (one of each tensor) a stage.
template <int DT, int NT, int NP, int VEC, int W, int S>
struct Rows {
  static constexpr int kRow = ring_row<W, NP, VEC>();
  const NormParams& p;
  Cols<W, VEC> c;
  uint32_t ring, bars;  // shared addresses: stages, S mbarriers
  int slot = 0;
  uint32_t ph = 0;
  bool ok = true;
  // VEC 1: the current row's offset in each tensor's blocks, by bytes, 64 added (the thread
  // that asks for a row leaves it beside the row); the top bit: not all in the ring
  uint32_t* codes;
  uint32_t code = 0;

  // Tensor k: forward y, x; backward r, dz, y, dr (null: not there, read as zero).  Addresses
  // stay in the kernel's parameters, not in registers.
  __device__ __forceinline__ const unsigned short* base(int k) const {
    const void* const t = NT == 2 ? (k == 0 ? p.y : p.x) : (k == 0 ? p.r : k == 1 ? p.dz : k == 2 ? p.y : p.dr);
    return static_cast<const unsigned short*>(t);
  }
  __device__ __forceinline__ long long ld(int k) const {
    return NT == 2 ? (k == 0 ? p.ldy : p.ldx) : (k == 0 ? p.ldr : k == 1 ? p.lddz : k == 2 ? p.ldy : p.lddr);
  }

  // Where row `row` of tensor k lies: the blocks copied [from, to) and the offset of column 0
  // in them (columns).
  struct Span {
    uintptr_t from;
    uint32_t bytes;
    int shift;
  };
  __device__ __forceinline__ Span span(int k, int row) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(base(k) + row * ld(k));
    if constexpr (VEC == 8) return {a, static_cast<uint32_t>(c.D) * 2, 0};
    const uintptr_t e = a + static_cast<uintptr_t>(c.D) * 2;
    uintptr_t from = a & ~static_cast<uintptr_t>(15), to = (e + 15) & ~static_cast<uintptr_t>(15);
    if (from < reinterpret_cast<uintptr_t>(base(k))) from += 16;
    if (to > reinterpret_cast<uintptr_t>(base(k) + (p.T - 1) * ld(k) + c.D)) to -= 16;
    const int shift = static_cast<int>(static_cast<intptr_t>(a - from)) / 2;
    return {from, to > from ? static_cast<uint32_t>(to - from) : 0u, shift};
  }
  // The ring starts as zeros: what no copy fills (columns past the row, absent tensors) stays so.
  __device__ __forceinline__ void init(uint8_t* smem, uint64_t* mbars, uint32_t* row_codes) {
    ring = smem_u32(smem), bars = smem_u32(mbars), codes = row_codes;
    if (VEC == 8 && NP * 2 * 32 * W != c.D) {
      for (int i = c.tid * 16; i < S * NT * kRow; i += 32 * W * 16) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
    } else if (VEC == 8 && base(NT - 1) == nullptr) {
      for (int i = c.tid * 16; i < S * NT * kRow; i += 32 * W * 16)
        if (i / kRow % NT == NT - 1) *reinterpret_cast<uint4*>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (c.tid == 0) {
      for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, 1);
      fence_mbar_init();
    }
    fence_proxy_async_smem();  // the zeros come before the copies
    __syncthreads();
  }
  // Asks for a row ahead of its use (row group's first thread).
  __device__ __forceinline__ void ask(int ahead, int row) {
    if (c.tid == 0 && ok) {
      const int at = slot + ahead >= S ? slot + ahead - S : slot + ahead;
      Span sp[NT];
      uint32_t bytes = 0;
#pragma unroll
      for (int k = 0; k < NT; ++k)
        if (base(k) != nullptr) sp[k] = span(k, row), bytes += sp[k].bytes;
      if constexpr (VEC == 1) {
        uint32_t v = 0;
        bool whole = true;
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          if (base(k) == nullptr) continue;
          v |= static_cast<uint32_t>(sp[k].shift + 64) << (8 * k);
          whole = whole && sp[k].shift >= 0 && static_cast<int>(sp[k].bytes / 2) - sp[k].shift >= c.D;
        }
        codes[at] = whole ? v : v | 0x80000000u;
      }
      mbar_arrive_expect_tx(bars + 8 * at, bytes);  // (releases the code with the row)
#pragma unroll
      for (int k = 0; k < NT; ++k)
        if (base(k) != nullptr && (VEC == 8 || sp[k].bytes > 0))
          bulk_load_g2s(ring + (at * NT + k) * kRow, reinterpret_cast<const void*>(sp[k].from), sp[k].bytes, bars + 8 * at);
    }
  }
  // Waits for the current stage's rows (bounded; once it ran out, no further wait).
  __device__ __forceinline__ void take() {
    if (ok && !mbar_wait(bars + 8 * slot, ph, p.timeout_ns, nullptr)) {
      ok = false;
      if (atomicCAS(p.status, 0, kStatusTimeout) == 0) {
        p.status[1] = 0x50;
        p.status[2] = static_cast<int>(blockIdx.x);
      }
      for (int i = 0; i < S; ++i)  // let the copies in flight land before the CTA can end
        mbar_wait(bars + 8 * ((slot + i) % S), ph ^ (slot + i >= S ? 1u : 0u), kDrainTimeoutNs, nullptr);
    }
    if constexpr (VEC == 1) code = ok ? codes[slot] : 0x40404040u;
  }
  __device__ __forceinline__ int shift(int k) const { return static_cast<int>((code >> (8 * k)) & 127u) - 64; }
  __device__ __forceinline__ void next() {
    if (++slot == S) slot = 0, ph ^= 1;
  }
  // Pairs e0 .. e0 + 3 of tensor k's row.
  __device__ __forceinline__ void get(int k, int row, int e0, Two (&f)[4]) const {
    const uint32_t at = ring + (slot * NT + k) * kRow;
    if constexpr (VEC == 8) {
      const uint4 q = lds128(at + c.first(e0) * 2);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2<DT>(w[i]);
        f[i] = two(v.x, v.y);
      }
    } else {
      if (base(k) == nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = two(0.f);
        return;
      }
      unsigned short raw[8];
      const uint32_t src = at + 2 * (c.tid + shift(k));
      if ((code & 0x80000000u) == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)  // in the ring's bounds for any column a thread holds
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw[i]) : "r"(src + (2 * e0 + i) * 64 * W) : "memory");
      } else {  // the tensor's first or last row: its first or last block is read directly
        const int hi = static_cast<int>(span(k, row).bytes / 2) - shift(k);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = c.tid + (2 * e0 + i) * 32 * W;
          raw[i] = 0;
          if (col < c.D) {
            if (col + shift(k) >= 0 && col < hi)
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw[i]) : "r"(src + (2 * e0 + i) * 64 * W) : "memory");
            else
              raw[i] = __ldg(base(k) + row * ld(k) + col);
          }
        }
      }
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = DT == DT_BF16 ? __bfloat162float(__ushort_as_bfloat16(raw[i])) : __half2float(__ushort_as_half(raw[i]));
        if (c.maybe_out(2 * e0 + i, NP)) v[i] = c.tid + (2 * e0 + i) * 32 * W < c.D ? v[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = two(v[2 * i], v[2 * i + 1]);
    }
  }
};

// Walks this CTA's units; a unit's rows go to its row groups in turn.  fn.unit(grp) at a
// unit's start, fn.row(row, ask) for each row, fn.done(u) at its end (the whole CTA calls it).
// A row's `ask` refills the slot of the row before: it is called after the row's first round
// of sums, when every warp is done with that one.
template <int W, int S, class R, class Fn>
__device__ __forceinline__ void walk(const NormParams& p, R& rows, Fn&& fn) {
  constexpr int RG = row_groups(W);
  for (int u = blockIdx.x; u < p.groups * p.chunks; u += gridDim.x) {
    const int grp = u / p.chunks, chunk = u - grp * p.chunks;
    const int lo = grp * p.rows_per_gate + chunk * RG + static_cast<int>(threadIdx.y);
    const int hi = (grp + 1) * p.rows_per_gate, by = p.chunks * RG;
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (lo + i * by < hi) rows.ask(i, lo + i * by);
    fn.unit(grp);
    for (int row = lo; row < hi; row += by) {
      rows.take();
      fn.row(row, [&] {
        if (row + (S - 1) * by < hi) rows.ask(S - 1, row + (S - 1) * by);
      });
      rows.next();
    }
    fn.done(u);
  }
}

// v - mean in the columns of the row, 0 past them.
template <int W, int VEC, int NP>
__device__ __forceinline__ void centre(Two (&v)[NP], float mean, const Cols<W, VEC>& c, int e0 = 0) {
  const Two m = two(-mean);
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const float2 f = both(add2(v[e], m));
    v[e] = two(c.in(e0 + e) ? f.x : 0.f, c.in2(e0 + e) ? f.y : 0.f);
  }
}

template <int DT, int W, int NP, int VEC, bool LAYER, int S>
struct FwdRow {
  const NormParams& p;
  Rows<DT, 2, NP, VEC, W, S>& in;  // y, x
  RowSum<W> sums;
  Two a[NP], w[NP];                                  // gate * w_post, w_pre
  Two b[LAYER ? NP : 1], bw[LAYER ? NP : 1];         // gate * b_post, b_pre

  __device__ __forceinline__ void unit(int grp) {
    const void* gate = p.gate == nullptr ? nullptr : vec_at(p.gate, p.vec_dtype, grp * p.ldgate);
    Two g[NP];
    load_param(gate, p.vec_dtype, in.c, 1.f, g);
    load_param(p.w_post, p.vec_dtype, in.c, 1.f, a);
    load_param(p.w_pre, p.vec_dtype, in.c, 1.f, w);
#pragma unroll
    for (int e = 0; e < NP; ++e) a[e] = mul2(a[e], g[e]);
    if constexpr (LAYER) {
      load_param(p.b_post, p.vec_dtype, in.c, 0.f, b);
      load_param(p.b_pre, p.vec_dtype, in.c, 0.f, bw);
#pragma unroll
      for (int e = 0; e < NP; ++e) b[e] = mul2(b[e], g[e]);
    }
  }
  __device__ __forceinline__ float rho(Two (&v)[NP], float inv) {  // v becomes v - mean in the LayerNorm form
    if constexpr (LAYER) {
      Two t = two(0.f);
#pragma unroll
      for (int e = 0; e < NP; ++e) t = add2(t, v[e]);
      float s[1] = {sum(t)};
      sums(s);
      centre(v, s[0] * inv, in.c);
    }
    Two t = two(0.f);
#pragma unroll
    for (int e = 0; e < NP; ++e) t = fma2(v[e], v[e], t);
    float q[1] = {sum(t)};
    sums(q);
    return rsqrtf(fmaf(q[0], inv, p.eps));
  }
  template <class Ask>
  __device__ __forceinline__ void row(int r, Ask&& ask) {
    const float inv = 1.0f / static_cast<float>(in.c.D);
    Two v[NP];
#pragma unroll
    for (int e0 = 0; e0 < NP; e0 += 4) {
      Two y[4];
      in.get(0, r, e0, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e0 + i] = y[i];
    }
    float k = 1.f;
    if (p.w_post != nullptr) {
      k = rho(v, inv);
      ask();
    }
    const Two k2 = two(k), sc = two(p.scale);
    unsigned short* rr = static_cast<unsigned short*>(p.r) + r * p.ldr;
#pragma unroll
    for (int e0 = 0; e0 < NP; e0 += 4) {
      Two x[4];
      in.get(1, r, e0, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i;
        if constexpr (LAYER) x[i] = fma2(sc, x[i], b[e]);
        else x[i] = mul2(sc, x[i]);
        v[e] = x[i] = fma2(mul2(v[e], k2), a[e], x[i]);
      }
      store_row<DT>(rr, in.c, e0, x);
    }
    k = rho(v, inv);
    if (p.w_post == nullptr) ask();
    const Two k3 = two(k);
    unsigned short* zr = static_cast<unsigned short*>(p.z) + r * p.ldz;
#pragma unroll
    for (int e0 = 0; e0 < NP; e0 += 4) {
      Two z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i;
        if constexpr (LAYER) z[i] = fma2(mul2(v[e], k3), w[e], bw[e]);
        else z[i] = mul2(mul2(v[e], k3), w[e]);
      }
      store_row<DT>(zr, in.c, e0, z);
    }
  }
  __device__ __forceinline__ void done(int) {}
};

// CTAs a SM: 64 registers a thread where it holds 4 pairs (80 in the LayerNorm form), else 128.
// 16384 x 4096 RMS: 92 us with 4 pairs and 32 warps a SM, 98 with 8 and 16; LayerNorm 153 and
// 115, but 77 and 107 at the odd width 1001.
constexpr int fwd_ctas(int W, int NP, bool layer) { return NP == 4 && !layer ? (W == 16 ? 2 : 4) : W == 16 ? 1 : NP == 4 ? 3 : 2; }

template <int DT, int W, int NP, int VEC, bool LAYER, int S>
__global__ void __launch_bounds__(32 * W * row_groups(W), NP == 8 ? 0 : fwd_ctas(W, NP, LAYER)) fo_norm_fwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int RG = row_groups(W);
  extern __shared__ __align__(128) uint8_t smem_norm[];
  __shared__ float red[RG * 2 * 16 * W];
  __shared__ __align__(8) uint64_t bars[RG * S];
  __shared__ uint32_t codes[RG * S];
  Rows<DT, 2, NP, VEC, W, S> in{p, {static_cast<int>(threadIdx.x), p.D}};
  in.init(smem_norm + threadIdx.y * S * 2 * in.kRow, bars + threadIdx.y * S, codes + threadIdx.y * S);
  FwdRow<DT, W, NP, VEC, LAYER, S> f{p, in, {red + threadIdx.y * 2 * 16 * W, 0, 1 + static_cast<int>(threadIdx.y)}, {}, {}, {}, {}};
  griddep_wait();
  griddep_launch_dependents();
  walk<W, S>(p, in, f);
}

template <int DT, int W, int NP, int VEC, bool LAYER>
struct BwdRow {
  static constexpr int kSums = LAYER ? 4 : 2;  // dz rhat, t yhat; and dz, t for the biases
  const NormParams& p;
  Rows<DT, 4, NP, VEC, W, kBwdStages>& in;  // r, dz, y, dr
  RowSum<W> sums;
  float* joint;  // [kSums][ldp] where the row groups of a CTA meet
  Two w[NP], a[NP];  // w_pre, gate * w_post
  Two acc[kSums][NP];

  __device__ __forceinline__ void unit(int grp) {
    const void* gate = p.gate == nullptr ? nullptr : vec_at(p.gate, p.vec_dtype, grp * p.ldgate);
    Two g[NP];
    load_param(gate, p.vec_dtype, in.c, 1.f, g);
    load_param(p.w_post, p.vec_dtype, in.c, 1.f, a);
    load_param(p.w_pre, p.vec_dtype, in.c, 0.f, w);
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      a[e] = mul2(a[e], g[e]);
#pragma unroll
      for (int k = 0; k < kSums; ++k) acc[k][e] = two(0.f);
    }
  }
  template <class Ask>
  __device__ __forceinline__ void row(int rw, Ask&& ask) {
    const float inv = 1.0f / static_cast<float>(in.c.D);
    const bool post = p.w_post != nullptr;
    float mr = 0.f, my = 0.f, mc = 0.f;
    // With 4 pairs a thread the row stays in registers; with 8 each pass reads the ring again.
    constexpr bool kHold = NP == 4;
    Two hr[4], hz[4], hy[4], hd[4];
    auto fetch = [&](int e0, Two (&r)[4], Two (&z)[4], Two (&y)[4], Two (&d)[4]) {
      if constexpr (kHold) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = hr[i], z[i] = hz[i], y[i] = hy[i], d[i] = hd[i];
      } else {
        in.get(0, rw, e0, r), in.get(1, rw, e0, z), in.get(2, rw, e0, y), in.get(3, rw, e0, d);
        if constexpr (LAYER) centre(r, mr, in.c, e0), centre(y, my, in.c, e0);
      }
    };
    if constexpr (kHold) in.get(0, rw, 0, hr), in.get(1, rw, 0, hz), in.get(2, rw, 0, hy), in.get(3, rw, 0, hd);
    if constexpr (LAYER) {
      Two s0 = two(0.f), s1 = s0, s2 = s0;
#pragma unroll
      for (int e0 = 0; e0 < NP; e0 += 4) {
        Two r[4], z[4], y[4];
        if constexpr (kHold) {
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] = hr[i], z[i] = hz[i], y[i] = hy[i];
        } else {
          in.get(0, rw, e0, r), in.get(1, rw, e0, z), in.get(2, rw, e0, y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s0 = add2(s0, r[i]), s1 = add2(s1, y[i]), s2 = fma2(z[i], w[e0 + i], s2);
      }
      float s[3] = {sum(s0), sum(s1), sum(s2)};
      sums(s);
      mr = s[0] * inv, my = post ? s[1] * inv : 0.f, mc = s[2] * inv;
      if constexpr (kHold) centre(hr, mr, in.c), centre(hy, my, in.c);
    }
    const Two mc2 = two(-mc);
    float kr, ky, m, me, me0 = 0.f;
    {
      // r^2, y^2, c r, A y dr, A y c, A y r, and in the LayerNorm form A dr, A c, A r
      Two t[6], l[3];
#pragma unroll
      for (int i = 0; i < 6; ++i) t[i] = two(0.f);
#pragma unroll
      for (int i = 0; i < 3; ++i) l[i] = two(0.f);
#pragma unroll
      for (int e0 = 0; e0 < NP; e0 += 4) {
        Two r[4], z[4], y[4], d[4];
        fetch(e0, r, z, y, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e0 + i;
          const Two ay = mul2(a[e], y[i]), c = LAYER ? fma2(z[i], w[e], mc2) : mul2(z[i], w[e]);
          t[0] = fma2(r[i], r[i], t[0]);
          t[1] = fma2(y[i], y[i], t[1]);
          t[2] = fma2(c, r[i], t[2]);
          t[3] = fma2(ay, d[i], t[3]);
          t[4] = fma2(ay, c, t[4]);
          t[5] = fma2(ay, r[i], t[5]);
          if constexpr (LAYER) {
            l[0] = fma2(a[e], d[i], l[0]);
            l[1] = fma2(a[e], c, l[1]);
            l[2] = fma2(a[e], r[i], l[2]);
          }
        }
      }
      float q[LAYER ? 9 : 6];
#pragma unroll
      for (int i = 0; i < 6; ++i) q[i] = sum(t[i]);
      if constexpr (LAYER) q[6] = sum(l[0]), q[7] = sum(l[1]), q[8] = sum(l[2]);
      sums(q);
      ask();
      kr = rsqrtf(fmaf(q[0], inv, p.eps)), ky = post ? rsqrtf(fmaf(q[1], inv, p.eps)) : 1.f;
      m = q[2] * inv * kr;  // mean(c rhat)
      // mean(e yhat) and mean(e) of e = A t, t = dr + kr c - kr kr m r
      me = post ? ky * inv * fmaf(kr, fmaf(-kr * m, q[5], q[4]), q[3]) : 0.f;
      if constexpr (LAYER) me0 = post ? inv * fmaf(kr, fmaf(-kr * m, q[8], q[7]), q[6]) : 0.f;
    }
    const Two kr2 = two(kr), ky2 = two(ky), nm = two(-m), nme = two(-me), sc = two(p.scale);
    const Two nme0 = two(-me0);
    unsigned short* dxr = static_cast<unsigned short*>(p.dx) + rw * p.lddx;
    unsigned short* dyr = static_cast<unsigned short*>(p.dy) + rw * p.lddy;
#pragma unroll
    for (int e0 = 0; e0 < NP; e0 += 4) {
      Two r[4], z[4], y[4], d[4], o[4];
      fetch(e0, r, z, y, d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i;
        const Two rh = mul2(r[i], kr2), yh = mul2(y[i], ky2);
        const Two c = LAYER ? fma2(z[i], w[e], mc2) : mul2(z[i], w[e]);
        const Two t = fma2(kr2, fma2(rh, nm, c), d[i]);
        acc[0][e] = fma2(z[i], rh, acc[0][e]);
        acc[1][e] = fma2(t, yh, acc[1][e]);
        if constexpr (LAYER) acc[2][e] = add2(acc[2][e], z[i]), acc[3][e] = add2(acc[3][e], t);
        d[i] = mul2(sc, t);
        Two q = fma2(yh, nme, mul2(a[e], t));
        if constexpr (LAYER) q = add2(q, nme0);
        o[i] = mul2(ky2, q);
      }
      store_row<DT>(dxr, in.c, e0, d);
      store_row<DT>(dyr, in.c, e0, o);
    }
  }
  __device__ __forceinline__ void done(int u) {
    constexpr int RG = row_groups(W);
    float* out = p.part + static_cast<long long>(u) * kSums * p.ldp;
#pragma unroll 1
    for (int g = 0; g < RG; ++g) {  // the row groups add up in turn, the last one writes
      if (g == static_cast<int>(threadIdx.y)) {
#pragma unroll
        for (int k = 0; k < kSums; ++k)
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            const float2 v = both(acc[k][e]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = k * p.ldp + (h ? in.c.second(e) : in.c.first(e));
              if (!(h ? in.c.in2(e) : in.c.in(e))) continue;
              const float t = (h ? v.y : v.x) + (g == 0 ? 0.f : joint[at]);
              if (g == RG - 1) out[at] = t;
              else joint[at] = t;
            }
          }
      }
      if (RG > 1) __syncthreads();
    }
  }
};

template <int DT, int W, int NP, int VEC, bool LAYER>
__global__ void __launch_bounds__(32 * W * row_groups(W), W == 16 ? 1 : 2) fo_norm_bwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int RG = row_groups(W), S = kBwdStages;
  extern __shared__ __align__(128) uint8_t smem_norm[];
  __shared__ float red[RG * 2 * 16 * W];
  __shared__ __align__(8) uint64_t bars[RG * S];
  __shared__ uint32_t codes[RG * S];
  Rows<DT, 4, NP, VEC, W, S> in{p, {static_cast<int>(threadIdx.x), p.D}};
  in.init(smem_norm + threadIdx.y * S * 4 * in.kRow, bars + threadIdx.y * S, codes + threadIdx.y * S);
  float* joint = reinterpret_cast<float*>(smem_norm + RG * S * 4 * in.kRow);
  BwdRow<DT, W, NP, VEC, LAYER> f{p, in, {red + threadIdx.y * 2 * 16 * W, 0, 1 + static_cast<int>(threadIdx.y)}, joint, {}, {}, {}};
  griddep_wait();
  griddep_launch_dependents();
  walk<W, S>(p, in, f);
}

// Joins the units' sums in a fixed order and forms the parameter gradients: block (output
// row, 32 columns).  Output rows 0..3 are dw_pre, dw_post, db_pre, db_post (all units), 4 + g
// the gate rows (their own chunks); where a gate row has one unit, and there are many of them,
// 4 + g stands for 32 gate rows, which a block only scales (4096 x 4096 bf16 RMS backward with
// a gate a token: 403 us; a block a row 2640).
struct JoinParams {
  const float* part;
  void* out[5];  // dw_pre, dw_post, db_pre, db_post, dgate; null: not wanted
  const void *w_post, *b_post, *gate;
  long long ldgate;
  int units, chunks, ldp, D, vec_dtype;
  int sums;  // a unit: BwdRow's kSums
};

constexpr int kJoinSplit = 32;

__global__ void __launch_bounds__(8 * kJoinSplit) fo_norm_join_kernel(const JoinParams p) {
  __shared__ float4 red[2][kJoinSplit][8];
  griddep_launch_dependents();
  griddep_wait();
  const int k = min(static_cast<int>(blockIdx.x), 4);
  if (p.out[k] == nullptr) return;
  const int g = static_cast<int>(blockIdx.x) - 4;
  auto store = [&](long long at, float v) {
    if (p.vec_dtype == DT_F32) static_cast<float*>(p.out[k])[at] = v;
    if (p.vec_dtype == DT_BF16) static_cast<__nv_bfloat16*>(p.out[k])[at] = __float2bfloat16_rn(v);
    if (p.vec_dtype == DT_F16) static_cast<__half*>(p.out[k])[at] = __float2half_rn(v);
  };
  // a gate row's gradient from its sums of t yhat and t
  auto of_gate = [&](int col, float ty, float t) {
    if (p.w_post != nullptr) ty *= load_vec(p.w_post, p.vec_dtype, col);
    return p.b_post != nullptr ? fmaf(load_vec(p.b_post, p.vec_dtype, col), t, ty) : ty;
  };
  if (k == 4 && p.chunks == 1) {
    const int row = g * kJoinSplit + static_cast<int>(threadIdx.x >> 3), col = static_cast<int>(blockIdx.y) * 32 + (threadIdx.x & 7) * 4;
    if (row >= p.units || col >= p.D) return;
    const float* src = p.part + (static_cast<long long>(row) * p.sums + 1) * p.ldp + col;
    const float4 q = __ldcg(reinterpret_cast<const float4*>(src));
    const float4 t = p.b_post != nullptr ? __ldcg(reinterpret_cast<const float4*>(src + 2 * static_cast<long long>(p.ldp))) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float ty[4] = {q.x, q.y, q.z, q.w}, ts[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < p.D) store(static_cast<long long>(row) * p.D + col + j, of_gate(col + j, ty[j], ts[j]));
    return;
  }
  const int lo = k < 4 ? 0 : g * p.chunks, hi = k < 4 ? p.units : lo + p.chunks;
  const int lane = threadIdx.x & 7, split = threadIdx.x >> 3;
  const int c = blockIdx.y * 32 + lane * 4;
  const bool gated = (k == 1 || k == 3) && p.gate != nullptr;  // sums weighted by each unit's gate row
  // dw_pre: dz rhat; dw_post, dgate: t yhat; db_pre: dz; db_post (and dgate's bias part): t
  const int slot = k == 0 ? 0 : k == 2 ? 2 : k == 3 ? 3 : 1;
  float a[2][4] = {};
  if (c < p.ldp) {
    const float* src = p.part + static_cast<long long>(slot) * p.ldp + c;
    int grp = -1;
    float gv[4] = {1.f, 1.f, 1.f, 1.f};
    for (int u0 = lo + split; u0 < hi; u0 += 4 * kJoinSplit) {  // four loads under way at once
      float4 q[4], t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + i * kJoinSplit;
        q[i] = t[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < hi) {
          q[i] = __ldcg(reinterpret_cast<const float4*>(src + static_cast<long long>(u) * p.sums * p.ldp));
          if (k == 4 && p.b_post != nullptr) t[i] = __ldcg(reinterpret_cast<const float4*>(src + (static_cast<long long>(u) * p.sums + 2) * p.ldp));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + i * kJoinSplit;
        if (gated && u < hi && u / p.chunks != grp) {
          grp = u / p.chunks;
          const void* row = vec_at(p.gate, p.vec_dtype, grp * p.ldgate);
#pragma unroll
          for (int j = 0; j < 4; ++j) gv[j] = c + j < p.D ? load_vec(row, p.vec_dtype, c + j) : 0.f;
        }
        a[0][0] = fmaf(q[i].x, gv[0], a[0][0]), a[0][1] = fmaf(q[i].y, gv[1], a[0][1]);
        a[0][2] = fmaf(q[i].z, gv[2], a[0][2]), a[0][3] = fmaf(q[i].w, gv[3], a[0][3]);
        a[1][0] += t[i].x, a[1][1] += t[i].y, a[1][2] += t[i].z, a[1][3] += t[i].w;
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) red[h][split][lane] = make_float4(a[h][0], a[h][1], a[h][2], a[h][3]);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int cc = blockIdx.y * 32 + threadIdx.x;
    float t = 0.f, t1 = 0.f;
#pragma unroll
    for (int s = 0; s < kJoinSplit; ++s) {
      t += reinterpret_cast<const float*>(red[0][s])[threadIdx.x];
      t1 += reinterpret_cast<const float*>(red[1][s])[threadIdx.x];
    }
    if (cc < p.D) {
      if (k == 4) t = of_gate(cc, t, t1);
      store((k < 4 ? 0 : static_cast<long long>(g) * p.D) + cc, t);
    }
  }
}

// ---------------------------------------------------------------------- host
using NormKernel = void (*)(const NormParams);

struct Shape {
  NormKernel kern;
  int warps, smem, ctas;
  std::atomic<uint64_t>* opted;
};

template <int DT, int W, int NP, int VEC, bool LAYER, int S = 4>
Shape fwd_entry(int) {
  static std::atomic<uint64_t> opted{0};
  return {fo_norm_fwd_kernel<DT, W, NP, VEC, LAYER, S>, W, row_groups(W) * S * 2 * ring_row<W, NP, VEC>(), fwd_ctas(W, NP, LAYER), &opted};
}

template <int DT, int W, int NP, int VEC, bool LAYER>
Shape bwd_entry(int D) {
  static std::atomic<uint64_t> opted{0};
  const int joint = row_groups(W) > 1 ? (LAYER ? 4 : 2) * ((D + 3) / 4 * 4) * 4 : 0;
  return {fo_norm_bwd_kernel<DT, W, NP, VEC, LAYER>, W, row_groups(W) * kBwdStages * 4 * ring_row<W, NP, VEC>() + joint, 2, &opted};
}

// The row layout for D columns: the fewest warps whose threads hold at most 8 pairs, or 4.
#define FO_NORM_SHAPES(entry, pairs4, vec)                 \
  if constexpr (!(pairs4)) {                               \
    if (D <= 256) return entry<DT, 1, 4, vec, LAYER>(D);   \
    if (D <= 512) return entry<DT, 1, 8, vec, LAYER>(D);   \
    if (D <= 1024) return entry<DT, 2, 8, vec, LAYER>(D);  \
    if (D <= 2048) return entry<DT, 4, 8, vec, LAYER>(D);  \
    if (D <= 4096) return entry<DT, 8, 8, vec, LAYER>(D);  \
  } else {                                                 \
    if (D <= 256) return entry<DT, 1, 4, vec, LAYER>(D);   \
    if (D <= 512) return entry<DT, 2, 4, vec, LAYER>(D);   \
    if (D <= 1024) return entry<DT, 4, 4, vec, LAYER>(D);  \
    if (D <= 2048) return entry<DT, 8, 4, vec, LAYER>(D);  \
    if (D <= 4096) return entry<DT, 16, 4, vec, LAYER>(D); \
  }

template <int DT, int VEC, bool LAYER>
Shape fwd_shape(int D) {
  FO_NORM_SHAPES(fwd_entry, !LAYER || VEC == 1, VEC)
  if (D <= 8192) return fwd_entry<DT, 16, 8, VEC, LAYER>(D);
  return fwd_entry<DT, 16, 16, VEC, LAYER, 3>(D);
}

template <int DT, int VEC, bool LAYER>
Shape bwd_shape(int D) {
  FO_NORM_SHAPES(bwd_entry, LAYER || VEC == 1, VEC)
  return bwd_entry<DT, 16, 8, VEC, LAYER>(D);
}

template <bool BWD, bool LAYER>
Shape shape_of(bool bf, bool v8, int D) {
  if constexpr (BWD) {
    if (bf) return v8 ? bwd_shape<DT_BF16, 8, LAYER>(D) : bwd_shape<DT_BF16, 1, LAYER>(D);
    return v8 ? bwd_shape<DT_F16, 8, LAYER>(D) : bwd_shape<DT_F16, 1, LAYER>(D);
  } else {
    if (bf) return v8 ? fwd_shape<DT_BF16, 8, LAYER>(D) : fwd_shape<DT_BF16, 1, LAYER>(D);
    return v8 ? fwd_shape<DT_F16, 8, LAYER>(D) : fwd_shape<DT_F16, 1, LAYER>(D);
  }
}

constexpr int kMaxFwd = 16384, kMaxBwd = 8192;
constexpr int64_t kMaxRows = 1ll << 30;  // rows ahead stay in 31 bits

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
  if (d->T > kMaxRows) return host_fail(FO_EINVAL, "T = %lld exceeds 2^30", static_cast<long long>(d->T));
  if (d->dtype != FO_DT_F16 && d->dtype != FO_DT_BF16) return host_fail(FO_EINVAL, "dtype must be FO_DT_F16 or FO_DT_BF16");
  if (d->vec_dtype < FO_DT_F16 || d->vec_dtype > FO_DT_F32) return host_fail(FO_EINVAL, "bad vec_dtype %d", d->vec_dtype);
  if (d->norm != FO_NORM_RMS && d->norm != FO_NORM_LAYER) return host_fail(FO_EINVAL, "norm must be FO_NORM_RMS or FO_NORM_LAYER");
  if (!(d->eps >= 0.f)) return host_fail(FO_EINVAL, "eps must be >= 0");
  if (d->w_post == nullptr && d->b_post != nullptr) return host_fail(FO_EINVAL, "b_post without w_post");
  if (d->norm == FO_NORM_RMS && (d->b_post != nullptr || d->b_pre != nullptr))
    return host_fail(FO_EINVAL, "the rms norm has no bias");
  if (bwd && d->norm == FO_NORM_RMS && (d->db_pre != nullptr || d->db_post != nullptr))
    return host_fail(FO_EINVAL, "the rms norm has no bias: db_pre and db_post must be null");
  if (bwd && d->w_post == nullptr && d->db_post != nullptr) return host_fail(FO_EINVAL, "db_post without w_post");
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

// Work split: units of rows inside one gate group, one a resident CTA (of 148 SMs, whatever the
// device: the backward workspace's size needs none); short batches give each row group one row
// at least.
struct Plan {
  int groups, chunks, units, ldp, sums;
  size_t bytes;  // of the units' sums: 8 (LayerNorm form: 16) a column of each
};

Plan plan(const FoBlockNormDesc* d, int per_sm, int row_groups) {
  Plan b{};
  const int cap = 148 * per_sm;
  b.groups = d->gate_rows > 0 ? static_cast<int>(d->gate_rows) : 1;
  const int rpg = static_cast<int>(d->T / b.groups);
  int chunks = b.groups >= cap ? 1 : cap / b.groups;
  const int turns = (rpg + row_groups - 1) / row_groups;
  if (chunks > turns) chunks = turns;
  if (chunks < 1) chunks = 1;
  b.chunks = chunks;
  b.units = b.groups * b.chunks;
  b.ldp = (static_cast<int>(d->D) + 3) / 4 * 4;
  b.sums = d->norm == FO_NORM_LAYER ? 4 : 2;
  b.bytes = static_cast<size_t>(b.units) * b.sums * b.ldp * sizeof(float);
  return b;
}

void set_plan(NormParams* p, const Plan& b) {
  p->groups = b.groups, p->chunks = b.chunks, p->ldp = b.ldp;
}

// The backward plan without a device, a dtype or addresses: the row groups of the 16-byte layout,
// and two CTAs a SM, one where the layout has 16 warps of 128 registers (LayerNorm 16384 x 4096
// 260 -> 243 us).
Plan bwd_plan(const FoBlockNormDesc* d) {
  const int W = d->D <= 512 ? 1 : d->D <= 1024 ? 2 : d->D <= 2048 ? 4 : 8;
  const bool wide = d->D > 4096 || (d->D > 2048 && (d->norm == FO_NORM_LAYER || d->D % 8 != 0));
  return plan(d, wide ? 1 : 2, kCtaWarps / W);
}

int min_grid(const Plan& b, int most) { return b.units < most ? b.units : most; }

std::atomic<uint64_t> g_no_opt{0};

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
  const Shape s = p.layer ? shape_of<false, true>(bf, v8, p.D) : shape_of<false, false>(bf, v8, p.D);
  const Plan b = plan(d, s.ctas, row_groups(s.warps));
  set_plan(&p, b);
  p.status = hd.status, p.timeout_ns = hd.timeout_ns;
  const cudaError_t e = launch_pdl(s.kern, *s.opted, dim3(min_grid(b, hd.sms * s.ctas)), dim3(32 * s.warps, row_groups(s.warps)), s.smem, 1,
                                   static_cast<cudaStream_t>(stream), p);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(1);
  return host_ok();
}

extern "C" size_t fo_block_norm_backward_workspace_size(const FoBlockNormDesc* d) {
  // sizes that the entry refuses ask for nothing (and may not fit the plan's integers)
  if (d == nullptr || d->T <= 0 || d->T > fo::kMaxRows || d->D <= 0 || d->D > fo::kMaxBwd || d->gate_rows < 0) return 0;
  if (d->gate_rows > 0 && d->T % d->gate_rows != 0) return 0;
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
  const Plan b = bwd_plan(d);
  if (d->workspace == nullptr || d->workspace_bytes < b.bytes || !host_aligned16(d->workspace))
    return host_fail(FO_EINVAL, "the backward pass needs a 16-byte aligned workspace of %zu bytes", b.bytes);
  HostDevice hd;
  if (int rc = host_device(&hd)) return rc;
  NormParams p;
  fill(&p, d);
  set_plan(&p, b);
  p.part = static_cast<float*>(d->workspace);
  p.status = hd.status, p.timeout_ns = hd.timeout_ns;
  const bool v8 = vectors(d, true), bf = d->dtype == FO_DT_BF16;
  const int D = p.D;
  const Shape s = p.layer ? shape_of<true, true>(bf, v8, D) : shape_of<true, false>(bf, v8, D);
  cudaError_t e = launch_pdl(s.kern, *s.opted, dim3(min_grid(b, hd.sms * 2)), dim3(32 * s.warps, row_groups(s.warps)), s.smem, 1, st, p);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  JoinParams j{};
  j.part = p.part;
  j.out[0] = d->dw_pre, j.out[1] = d->w_post != nullptr ? d->dw_post : nullptr, j.out[2] = d->db_pre, j.out[3] = d->db_post;
  j.out[4] = d->gate != nullptr ? d->dgate : nullptr;
  j.w_post = d->w_post, j.b_post = d->b_post, j.gate = d->gate, j.ldgate = d->ldgate;
  j.units = b.units, j.chunks = b.chunks, j.ldp = b.ldp, j.sums = b.sums, j.D = D, j.vec_dtype = d->vec_dtype;
  const unsigned rows = b.chunks == 1 ? static_cast<unsigned>((b.groups + kJoinSplit - 1) / kJoinSplit) : static_cast<unsigned>(b.groups);
  const unsigned outs = 4u + (d->gate != nullptr ? rows : 0u);
  e = launch_pdl(fo_norm_join_kernel, g_no_opt, dim3(outs, (D + 31) / 32), dim3(8 * kJoinSplit), 0, 1, st, j);
  if (e != cudaSuccess) return host_fail(FO_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
  host_count_launches(2);
  return host_ok();
}
