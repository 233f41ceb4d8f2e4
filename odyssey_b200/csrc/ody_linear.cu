// ody_linear.cu -- the linear layer over what the update step emits: products
// with the 4-bit weights as they lie, activations kept in 8 bits, and the
// weight gradient taken from them.
//
//   forward  y[m, n]  = s sum_k x[m, k] W[n, k]
//   dgrad    dx[m, k] = s sum_n dy[m, n] W[n, k]
//   wgrad    dW[n, k] = s sum_m dy[m, n] x'[m, k]  (+ add[n, k])
//
// W lies in the blocks of the flattened [out, in] weight (17 bytes for 32
// elements, 9 for 16), so a block may straddle two rows.  x' are 8-bit codes
// in rows of whole 32-column groups with one power of two per group.
#include "ody_linear.h"
#include "ody_linear_dev.cuh"
#include "ody_linear_gemm.h"
#include "ody_linear_rows.h"

namespace ody {

// ---------------------------------------------------------------------------
// Medium products, in one launch and without a workspace: 64 x 64 results per
// cluster of up to eight CTAs that share the reduction; 64 of the reduction
// at a time come through registers (the next 64 under way meanwhile), are
// brought to bfloat16 exactly, x or dy as one to three parts, and go through
// shared memory and ldmatrix to mma.sync.m16n8k16, eight warps with 16 x 32
// results each.  Below a few hundred rows this beats the tcgen05 kernel,
// whose operands have to be brought to bfloat16 by launches of their own and
// whose 256 x 256 tiles leave most SMs idle; the legacy tensor instruction
// has no tile to fill and its operands come straight from the decoding
// threads.  (The same tile on the FP32 pipe took 3.6 us for 64 of the
// reduction.)
//
// An operand's tile lies in shared memory as it does in memory, rows of 64
// elements at 144 bytes (nine 16-byte words: ldmatrix reads eight rows
// without a bank conflict); where those rows are the reduction's the
// fragments are read transposed.  Every 512 products the sums are added in
// float32 with rounding, as in the tcgen05 kernel.
// ---------------------------------------------------------------------------
constexpr int kMT = 64, kMPitch = 144, kMTile = kMT * kMPitch, kMSumPitch = kMT + 4;

// eight elements of x or dy as they lie in memory
template <int DT>
struct Eight {
  uint4 raw[DT == DT_F32 ? 2 : 1];
  // from element `at` of p; n of them are there; wide: they are 16-byte aligned
  __device__ __forceinline__ void load(const void* p, int64_t at, int n, bool wide) {
    if (wide && n >= 8) {
      const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + at * (DT == DT_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < (DT == DT_F32 ? 2 : 1); i++) raw[i] = __ldg(s + i);
    } else {
      uint32_t w[DT == DT_F32 ? 8 : 4] = {};
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) {
          if constexpr (DT == DT_F32)
            w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + at + i);
          else
            w[i >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + at + i) << (16 * (i & 1));
        }
#pragma unroll
      for (int i = 0; i < (DT == DT_F32 ? 2 : 1); i++) raw[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  // its parts, one tile each; a part is what the ones before it, cut to
  // bfloat16's bits, leave (after an infinity NaN)
  __device__ __forceinline__ void store(uint8_t* d) const {
    if constexpr (DT == DT_BF16) {
      *reinterpret_cast<uint4*>(d) = raw[0];
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint4& u = raw[DT == DT_F32 ? i >> 2 : 0];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        v[i] = DT == DT_F32 ? __uint_as_float(w[i & 3]) : f16_bits_to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
      }
#pragma unroll
      for (int p = 0; p < bf16_parts(DT); p++) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
        *reinterpret_cast<uint4*>(d + p * kMTile) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __fsub_rn(v[i], __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u));
      }
    }
  }
};

// Eight neighbouring elements of the quantised operand: codes in their order
// (weight i in nibble i ^ 1), scales, and as bfloat16.  Weights of rows that
// are not a multiple of eight wide may begin at any nibble and reach into a
// second block.
template <int OP, int KIND>
struct EightQ {
  uint32_t code[OP == LIN_WGRAD ? 2 : 1], scale;  // scale: of the elements before `split`, and 8 bits up the others'
  int split;
  // row r, column c; n elements are there (8 where blocks)
  __device__ __forceinline__ void load(const LinearArgs& p, int64_t groups, int64_t r, int64_t c, int n, bool blocks) {
    split = 8;
    if constexpr (OP == LIN_WGRAD) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p.q + r * groups * kA8Group + c));
      code[0] = u.x, code[1] = u.y;
      scale = __ldg(p.scales + r * groups + c / kA8Group);
    } else {
      using W = W4<KIND>;
      const uint64_t e = (uint64_t)(r * p.in + c);
      const uint8_t* const blk = p.q + e / W::BE * W::SB;
      const int i0 = (int)(e % W::BE);
      if (blocks) {
        const uint8_t* const s = blk + i0 / 2;
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = __ldg(s + i);
        scale = __ldg(blk + W::SB - 1);
        code[0] = u[0] | u[1] << 8 | u[2] << 16 | u[3] << 24;
      } else {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int j = i0 + i;
          u[i] = i < n ? __ldg(blk + (j < W::BE ? j / 2 : W::SB + (j - W::BE) / 2)) : 0u;
        }
        split = W::BE - i0;
        scale = __ldg(blk + W::SB - 1);
        if (split < n) scale |= (uint32_t)__ldg(blk + 2 * W::SB - 1) << 8;
        code[0] = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) code[0] |= (u[i] >> (i0 + i & 1 ? 0 : 4) & 15u) << (4 * (i ^ 1));
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* d) const {
    uint32_t o[4];
    if constexpr (OP == LIN_WGRAD) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t two = code[i >> 1] >> (16 * (i & 1));
        o[i] = __byte_perm(__float_as_uint(a8_value<KIND>(two & 255u, scale)),
                           __float_as_uint(a8_value<KIND>((two >> 8) & 255u, scale)), 0x7632);
      }
    } else {
      w4_raw8<KIND>(code[0], o);
      const uint32_t f0 = w4_scale_bf16x2<KIND>(scale & 255u), f1 = w4_scale_bf16x2<KIND>(scale >> 8 & 255u);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t f = 2 * i + 1 < split ? f0 : (2 * i >= split ? f1 : __byte_perm(f0, f1, 0x5410));
        o[i] = mul_bf16x2(mul_bf16x2(o[i], kTwo126), f);
      }
    }
    *reinterpret_cast<uint4*>(d) = make_uint4(o[0], o[1], o[2], o[3]);
  }
};

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t r[4]) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

template <int OP, int KIND, int DT>
__global__ void __launch_bounds__(256) medium_kernel(const LinearArgs p) {
  constexpr int P = bf16_parts(DT), STAGE = (P + 1) * kMTile;
  constexpr bool AR = OP != LIN_WGRAD, BR = OP == LIN_FORWARD;  // the contiguous axis is the reduction's
  extern __shared__ __align__(16) uint8_t medium_sm[];
  const int64_t M = OP == LIN_WGRAD ? p.out : p.rows, N = OP == LIN_FORWARD ? p.out : p.in;
  const int64_t R = OP == LIN_FORWARD ? p.in : (OP == LIN_DGRAD ? p.out : p.rows);
  const int64_t tn = (N + kMT - 1) / kMT, tile = blockIdx.x / cluster_size();
  const int64_t m0 = tile / tn * kMT, n0 = tile % tn * kMT;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const int64_t steps = (R + kMT - 1) / kMT, s0 = steps * rank / ranks, s1 = steps * (rank + 1) / ranks;
  const int64_t groups = (p.in + kA8Group - 1) / kA8Group;
  const bool blocks = OP == LIN_WGRAD || p.in % 8 == 0;  // eight columns share a block
  const bool wide = (reinterpret_cast<uintptr_t>(p.a) & 15u) == 0 && p.lda * (DT == DT_F32 ? 4 : 2) % 16 == 0;
  // this thread's part of a tile: eight elements of rows t / 8 and t / 8 + 32
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, row = t >> 3, col = (t & 7) * 8;
  uint8_t* const mine = medium_sm + row * kMPitch + col * 2;
  Eight<DT> a[2];
  EightQ<OP, KIND> b[2];
  bool on[2];
  const auto load = [&](int64_t s) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      // an operand's row and its column there
      const int64_t ar = (AR ? m0 : s * kMT) + row + 32 * i, ac = (AR ? s * kMT : m0) + col;
      a[i].load(p.a, ar * p.lda + ac, ar < (AR ? M : R) ? (int)max((int64_t)0, min((int64_t)8, (AR ? R : M) - ac)) : 0, wide);
      const int64_t br = (BR ? n0 : s * kMT) + row + 32 * i, bc = (BR ? s * kMT : n0) + col;
      on[i] = br < (BR ? N : R) && bc < p.in;
      if (on[i]) b[i].load(p, groups, br, bc, (int)min((int64_t)8, p.in - bc), blocks);
    }
  };
  const auto store = [&](int to) {
    uint8_t* const d = mine + to * STAGE;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      a[i].store(d + 32 * i * kMPitch);
      uint8_t* const e = d + P * kMTile + 32 * i * kMPitch;
      if (on[i])
        b[i].store(e);
      else
        *reinterpret_cast<uint4*>(e) = make_uint4(0, 0, 0, 0);
    }
  };
  // warp w: rows 16 (w % 4), columns 32 (w / 4) of the tile
  const int wm = (warp & 3) * 16, wn = (warp >> 2) * 32;
  // the eight-element row that this lane hands to ldmatrix, for k 0..15:
  // A's four 8 x 8 are (m, k), (m + 8, k), (m, k + 8), (m + 8, k + 8), B's
  // (n, k), (n, k + 8), (n + 8, k), (n + 8, k + 8)
  const int l8 = lane & 7, l16 = lane >> 3 & 1, l32 = lane >> 4;
  const uint32_t base = srow(medium_sm);
  const uint32_t af = base + (AR ? (wm + l8 + 8 * l16) * kMPitch + l32 * 16 : (l8 + 8 * l32) * kMPitch + (wm + 8 * l16) * 2);
  const uint32_t bf = base + P * kMTile +
                      (BR ? (wn + l8 + 8 * l32) * kMPitch + l16 * 16 : (l8 + 8 * l16) * kMPitch + (wn + 8 * l32) * 2);
  float acc[4][4] = {}, part[4][4] = {};
  load(s0);
  store(0);
  __syncthreads();
#pragma unroll 1
  for (int64_t s = s0; s < s1; s++) {
    const int to = (int)(s - s0) & 1;
    if (s + 1 < s1) load(s + 1);
#pragma unroll 2
    for (int k = 0; k < kMT; k += 16) {
      uint32_t x[4], y[2][4];
#pragma unroll
      for (int j = 0; j < 2; j++) ldmatrix4<!BR>(bf + to * STAGE + (BR ? k * 2 + j * 16 * kMPitch : k * kMPitch + j * 32), y[j]);
#pragma unroll
      for (int q = 0; q < P; q++) {
        ldmatrix4<!AR>(af + to * STAGE + q * kMTile + (AR ? k * 2 : k * kMPitch), x);
#pragma unroll
        for (int j = 0; j < 4; j++) mma16816(part[j], x[0], x[1], x[2], x[3], y[j >> 1][2 * (j & 1)], y[j >> 1][2 * (j & 1) + 1]);
      }
    }
    if (((s - s0) & 7) == 7 || s + 1 == s1) {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __fadd_rn(acc[i][j], part[i][j]), part[i][j] = 0.0f;
    }
    if (s + 1 < s1) store(to ^ 1);
    __syncthreads();
  }
  // every CTA's sums in shared memory; each adds and stores its share
  float* const red = reinterpret_cast<float*>(medium_sm);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float* d = red + (wm + (lane >> 2)) * kMSumPitch + wn + 8 * j + 2 * (lane & 3);
    d[0] = acc[j][0], d[1] = acc[j][1];
    d[8 * kMSumPitch] = acc[j][2], d[8 * kMSumPitch + 1] = acc[j][3];
  }
  const float scale = out_scale(p.o);
  if (ranks > 1)
    cluster_barrier();
  else
    __syncthreads();
#pragma unroll 2
  for (int o = rank * 256 + t; o < kMT * kMT; o += ranks * 256) {
    const int i = o / kMT, j = o % kMT;
    float v[8];
    if (ranks == 1) {
      v[0] = red[i * kMSumPitch + j];
    } else {
#pragma unroll
      for (uint32_t r = 0; r < 8; r++) v[r] = r < ranks ? peer_float(red + i * kMSumPitch + j, r) : 0.0f;
#pragma unroll
      for (uint32_t r = 1; r < 8; r++) v[0] = __fadd_rn(v[0], v[r]);
    }
    if (m0 + i < M && n0 + j < N) finish(p.o, scale, m0 + i, n0 + j, v[0]);
  }
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

static int lin_sms() {
  static int n[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] ? n[dev] : 148;
}

struct MediumPlan {
  int64_t tiles, steps;
  int ranks;
  int64_t rounds;  // steps that an SM with the most of them does one after another
};
static MediumPlan medium_plan(const LinearArgs& a, int sms) {
  const int64_t M = a.op == LIN_WGRAD ? a.out : a.rows, N = a.op == LIN_FORWARD ? a.out : a.in;
  const int64_t R = a.op == LIN_FORWARD ? a.in : (a.op == LIN_DGRAD ? a.out : a.rows);
  MediumPlan p;
  p.tiles = ((M + kMT - 1) / kMT) * ((N + kMT - 1) / kMT);
  p.steps = (R + kMT - 1) / kMT;
  p.ranks = 1;
  while (p.ranks < 8 && p.tiles * p.ranks * 2 <= 2 * sms && p.ranks < p.steps) p.ranks *= 2;
  const int64_t ctas = p.tiles * p.ranks;
  p.rounds = ((ctas + sms - 1) / sms) * ((p.steps + p.ranks - 1) / p.ranks);
  return p;
}

template <int OP, int KIND, int DT>
static cudaError_t launch_medium(const LinearArgs& a, const MediumPlan& p, cudaStream_t st) {
  constexpr int smem = 2 * (bf16_parts(DT) + 1) * kMTile;
  static_assert(smem >= kMT * kMSumPitch * 4, "the sums fit");
  static bool set[64] = {false};  // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(medium_kernel<OP, KIND, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  if (p.ranks == 1) {
    medium_kernel<OP, KIND, DT><<<(unsigned)p.tiles, 256, smem, st>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.tiles * p.ranks));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.ranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, medium_kernel<OP, KIND, DT>, a);
}

template <int OP, int KIND>
static cudaError_t launch_medium_dt(const LinearArgs& a, const MediumPlan& p, cudaStream_t st) {
  if (a.a_dtype == DT_F32) return launch_medium<OP, KIND, DT_F32>(a, p, st);
  if (a.a_dtype == DT_F16) return launch_medium<OP, KIND, DT_F16>(a, p, st);
  return launch_medium<OP, KIND, DT_BF16>(a, p, st);
}

template <int OP>
static cudaError_t launch_medium_w4(const LinearArgs& a, const MediumPlan& p, cudaStream_t st) {
  if (a.kind == Q_MXFP4) return launch_medium_dt<OP, Q_MXFP4>(a, p, st);
  if (a.kind == Q_MXFP4_OCP) return launch_medium_dt<OP, Q_MXFP4_OCP>(a, p, st);
  return launch_medium_dt<OP, Q_NVFP4>(a, p, st);  // the tensor scale of ODY_Q_NVFP4_TENSOR is applied to the sums
}

// Which way a product goes: few rows of whole blocks in one pass over the
// weight, medium ones in one launch, the others to the tcgen05 kernel after
// their operands have been brought to bfloat16.  The medium kernel takes 4 us
// and 0.9 us (float32 1.4) for each 64 of the reduction that an SM does; the
// other's launches take 15 us (16 with an operand to be split): 512 x 1024 x
// 1024 in bfloat16, 16 rounds, 17.4 us against 15.8; 256 x 1024 x 1024, 8
// rounds, 10.3 against 15.7.
constexpr int64_t kMediumRounds = 12;
static bool medium_product(const LinearArgs& a) { return medium_plan(a, lin_sms()).rounds <= kMediumRounds; }

// (of any kind: the query does not name one, so widths are taken to be in 32s)
int64_t linear_workspace(const LinearArgs& a) {
  return medium_product(a) || (few_rows(a) && a.in % 32 == 0) ? 0 : gemm_workspace(a, lin_sms());
}

cudaError_t launch_linear(const LinearArgs& a, void* ws, cudaStream_t st) {
  const int sms = lin_sms();
  if (few_rows(a)) return launch_few_rows(a, sms, st);
  const MediumPlan p = medium_plan(a, sms);
  if (p.rounds > kMediumRounds) return launch_gemm(a, ws, sms, st);
  if (a.op == LIN_FORWARD) return launch_medium_w4<LIN_FORWARD>(a, p, st);
  if (a.op == LIN_DGRAD) return launch_medium_w4<LIN_DGRAD>(a, p, st);
  return a.kind == A8_E4M3 ? launch_medium_dt<LIN_WGRAD, A8_E4M3>(a, p, st) : launch_medium_dt<LIN_WGRAD, A8_E5M2>(a, p, st);
}

// ---------------------------------------------------------------------------
// 8-bit activations.  Per row and 32 columns: X = the least power of two with
// amax <= largest * 2^X over the finite elements (largest = 448 = 1.75 * 2^8,
// or 57344 = 1.75 * 2^15), so no finite element saturates while X is inside
// its range; codes are RN(x * 2^-X), and the multiplication is exact wherever
// the code is not zero.  X stays where 2^X times every code is a normal
// bfloat16: the product of code and scale is then exact in both bfloat16 and
// float32.  Infinities must survive, since the step's finite check looks for
// them in the gradients made from these codes: E5M2 keeps them, E4M3 has none
// and stores NaN.
// ---------------------------------------------------------------------------
template <int FMT>
struct A8 {
  static constexpr int TOP = FMT == A8_E4M3 ? 8 : 15;
  static constexpr int XMIN = FMT == A8_E4M3 ? -117 : -110, XMAX = FMT == A8_E4M3 ? 119 : 112;
  static __device__ __forceinline__ int exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127 - TOP + ((b & 0x7fffffu) > 0x600000u);
    return x < XMIN ? XMIN : (x > XMAX ? XMAX : x);  // subnormal amax: below XMIN anyway
  }
  static __device__ __forceinline__ uint32_t encode(float x, float inv) {
    const uint32_t sign = (__float_as_uint(x) >> 24) & 0x80u;
    if (fabsf(x) == __uint_as_float(0x7f800000u)) return sign | (FMT == A8_E4M3 ? 0x7fu : 0x7cu);
    const float v = __fmul_rn(x, inv);
    return FMT == A8_E4M3 ? f32_to_e4m3(v) : f32_to_e5m2(v);
  }
};

// Four lanes share a group, eight elements each: two 16-byte loads of float32
// or one of 16-bit elements where the row's alignment allows it.
template <int FMT, int DT>
__global__ void __launch_bounds__(256) act8_save_kernel(const void* x, int64_t rows, int64_t cols, int64_t ldx,
                                                        uint8_t* codes, uint8_t* scales, int wide) {
  const int64_t groups = (cols + kA8Group - 1) / kA8Group;
  const int64_t total = rows * groups * 4;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < (total + 31) / 32 * 32; t += stride) {
    float v[8] = {};
    const bool on = t < total;
    const int64_t g = t >> 2, row = on ? g / groups : 0;
    const int64_t c0 = (g - row * groups) * kA8Group + (t & 3) * 8;
    if (on) {
      const int64_t at = row * ldx + c0;
      if (wide && c0 + 8 <= cols) {
        if (DT == DT_F32) {
          const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + at);
          const float4 a = __ldcs(s), b = __ldcs(s + 1);
          v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
          const uint4 u = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + at));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            v[2 * i] = DT == DT_F16 ? f16_bits_to_f32(w[i] & 0xffff) : bf16_bits_to_f32(w[i] & 0xffff);
            v[2 * i + 1] = DT == DT_F16 ? f16_bits_to_f32(w[i] >> 16) : bf16_bits_to_f32(w[i] >> 16);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (c0 + i < cols) v[i] = load_elem(x, DT, at + i);
      }
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float a = fabsf(v[i]);
      amax = a < __uint_as_float(0x7f800000u) ? fmaxf(amax, a) : amax;  // finite elements only
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (!on) continue;
    const int ex = A8<FMT>::exponent(amax);
    const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      lo |= A8<FMT>::encode(v[i], inv) << (8 * i);
      hi |= A8<FMT>::encode(v[4 + i], inv) << (8 * i);
    }
    __stcs(reinterpret_cast<uint2*>(codes) + t, make_uint2(lo, hi));
    if ((t & 3) == 0) scales[g] = (uint8_t)(ex + 127);
  }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(256) act8_load_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                        int64_t cols, void* out, int64_t ldo, int wide) {
  const int64_t groups = (cols + kA8Group - 1) / kA8Group;
  const int64_t total = rows * groups * 4;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < total; t += stride) {
    const int64_t g = t >> 2, row = g / groups;
    const int64_t c0 = (g - row * groups) * kA8Group + (t & 3) * 8;
    if (c0 >= cols) continue;
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(codes) + t);
    const uint32_t sb = scales[g];
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[i] = a8_value<FMT>((w.x >> (8 * i)) & 255u, sb);
      v[4 + i] = a8_value<FMT>((w.y >> (8 * i)) & 255u, sb);
    }
    if (DT == DT_F16) {
      // a finite value that rounded past float16's largest stays finite (it
      // came from a finite element); an infinity stays one
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (fabsf(v[i]) < __uint_as_float(0x7f800000u)) v[i] = fminf(fmaxf(v[i], -65504.0f), 65504.0f);
    }
    const int64_t at = row * ldo + c0;
    if (wide && c0 + 8 <= cols) {
      if (DT == DT_F32) {
        float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
        __stcs(d, make_float4(v[0], v[1], v[2], v[3]));
        __stcs(d + 1, make_float4(v[4], v[5], v[6], v[7]));
      } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
          u[i] = DT == DT_F16 ? f32_to_f16_bits(v[2 * i]) | (uint32_t)f32_to_f16_bits(v[2 * i + 1]) << 16
                              : f32_to_bf16_bits(v[2 * i]) | (uint32_t)f32_to_bf16_bits(v[2 * i + 1]) << 16;
        __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at), make_uint4(u[0], u[1], u[2], u[3]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c0 + i < cols) store_elem(out, DT, at + i, v[i]);
    }
  }
}

static int act8_grid(int64_t rows, int64_t cols) {
  const int64_t want = (rows * ((cols + kA8Group - 1) / kA8Group) * 4 + 255) / 256;
  const int64_t cap = (int64_t)lin_sms() * 32;
  return (int)(want < cap ? want : cap);
}

// whether 16-byte accesses at multiples of eight columns are aligned
static int wide_rows(const void* p, int dtype, int64_t ld) {
  const int64_t e = dtype == DT_F32 ? 4 : 2;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * e) % 16 == 0;
}

cudaError_t launch_act8_save(int fmt, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                             uint8_t* scales, cudaStream_t st) {
  const int grid = act8_grid(rows, cols), w = wide_rows(x, dtype, ldx);
#define ODY_S(F, D) \
  if (fmt == F && dtype == D) act8_save_kernel<F, D><<<grid, 256, 0, st>>>(x, rows, cols, ldx, codes, scales, w);
  ODY_S(A8_E4M3, DT_F32) ODY_S(A8_E4M3, DT_F16) ODY_S(A8_E4M3, DT_BF16)
  ODY_S(A8_E5M2, DT_F32) ODY_S(A8_E5M2, DT_F16) ODY_S(A8_E5M2, DT_BF16)
#undef ODY_S
  return cudaGetLastError();
}

cudaError_t launch_act8_load(int fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                             int dtype, int64_t ldo, cudaStream_t st) {
  const int grid = act8_grid(rows, cols), w = wide_rows(out, dtype, ldo);
#define ODY_L(F, D) \
  if (fmt == F && dtype == D) act8_load_kernel<F, D><<<grid, 256, 0, st>>>(codes, scales, rows, cols, out, ldo, w);
  ODY_L(A8_E4M3, DT_F32) ODY_L(A8_E4M3, DT_F16) ODY_L(A8_E4M3, DT_BF16)
  ODY_L(A8_E5M2, DT_F32) ODY_L(A8_E5M2, DT_F16) ODY_L(A8_E5M2, DT_BF16)
#undef ODY_L
  return cudaGetLastError();
}

}  // namespace ody
