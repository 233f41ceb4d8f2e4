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
// fragments are read transposed.  Every 32 mma the sums are added in float32
// with rounding, as in the tcgen05 kernel.
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
  constexpr int P = bf16_parts(DT), STAGE = (P + 1) * kMTile, KEEP = 8 / P;  // steps of 4 P mma in one sum
  constexpr bool AR = OP != LIN_WGRAD, BR = OP == LIN_FORWARD;  // the contiguous axis is the reduction's
  extern __shared__ __align__(16) uint8_t medium_sm[];
  const int64_t M = OP == LIN_WGRAD ? p.out : p.rows, N = OP == LIN_FORWARD ? p.out : p.in;
  const int64_t R = OP == LIN_FORWARD ? p.in : (OP == LIN_DGRAD ? p.out : p.rows);
  const int64_t tn = (N + kMT - 1) / kMT, tile = blockIdx.x / cluster_size();
  const int64_t m0 = tile / tn * kMT, n0 = tile % tn * kMT;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const int64_t steps = (R + kMT - 1) / kMT, s0 = steps * rank / ranks, s1 = steps * (rank + 1) / ranks;
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
      if (on[i]) b[i].load(p.q, p.scales, p.in, br, bc, (int)min((int64_t)8, p.in - bc), blocks);
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
    if ((s - s0) % KEEP == KEEP - 1 || s + 1 == s1) {
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
  static std::atomic<int> known[kMaxDevices];
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return 148;
  if ((n = known[dev].load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
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
  static PerDevice set;
  if (const cudaError_t e = allow_shared(set, (const void*)medium_kernel<OP, KIND, DT>, smem)) return e;
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
// and about 1 us (float32 1.3) for each 64 of the reduction that an SM does,
// the others start at 14 us (18 with an operand to be split).  512 x 1024 x
// 1024, 16 rounds: 20.3 us against 15.3 in bfloat16, 25.6 against 19.1 in
// float32; 256 x 1024 x 1024, 8 rounds: 12.0 against 14.4, 14.7 against 18.4.
// The few-row kernels take all that their registers hold: 32 rows x 8192^2
// forward 34 us, by the tcgen05 kernel 68; 16 rows backward 29 against 66; 5
// rows x 1024^2 forward 3.8 us, by the medium kernel 7.4.  (Small products of
// several float32 rows would gain there, 4 x 128 x 384 5.1 us for 7.9; they
// stay, since among few rows a row's results then do not depend on how many
// there are.)
constexpr int64_t kMediumRounds = 12;
static bool medium_product(const LinearArgs& a) { return medium_plan(a, lin_sms()).rounds <= kMediumRounds; }

int64_t linear_workspace(const LinearArgs& a) { return few_rows(a) || medium_product(a) ? 0 : gemm_workspace(a, lin_sms()); }

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
  // the power for a finite amax (its bits); subnormal ones are below XMIN anyway
  static __device__ __forceinline__ int exponent(uint32_t amax) {
    const int x = (int)(amax >> 23) - 127 - TOP + ((amax & 0x7fffffu) > 0x600000u);
    return min(max(x, XMIN), XMAX);
  }
  static __device__ __forceinline__ uint32_t encode(float x, float inv) {
    const uint32_t sign = (__float_as_uint(x) >> 24) & 0x80u;
    if (fabsf(x) == __uint_as_float(0x7f800000u)) return sign | (FMT == A8_E4M3 ? 0x7fu : 0x7cu);
    const float v = __fmul_rn(x, inv);
    return FMT == A8_E4M3 ? f32_to_e4m3(v) : f32_to_e5m2(v);
  }
  // two finite values; the first in the low byte
  static __device__ __forceinline__ uint32_t encode2(float x, float y, float inv) {
    return __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x, inv), __fmul_rn(y, inv)), __NV_SATFINITE,
                                    FMT == A8_E4M3 ? __NV_E4M3 : __NV_E5M2);
  }
};

// Both directions move 1 + 1/32 bytes a value on one side and the value on
// the other, so they are bound by memory; a thread has four runs of eight
// values under way, and what it does to them is counted: the largest
// magnitude of 16-bit values is found on their bits, two at a time, values
// are converted in pairs, and only a warp that meets a NaN or infinity looks
// at single elements (8192 x 4096 in bfloat16: element by element 37 us).
constexpr int kRuns = 4;

// eight elements: the bits as they lie, their largest magnitude (as the bits
// of a float32), and as float32
template <int DT>
struct Run8 {
  uint4 raw[DT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* x, int64_t at, int n, bool wide) {
    if (wide && n >= 8) {
      const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(x) + at * (DT == DT_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < (DT == DT_F32 ? 2 : 1); i++) raw[i] = __ldcs(s + i);
    } else {
      uint32_t w[DT == DT_F32 ? 8 : 4] = {};
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) {
          if constexpr (DT == DT_F32)
            w[i] = __ldg(reinterpret_cast<const uint32_t*>(x) + at + i);
          else
            w[i >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(x) + at + i) << (16 * (i & 1));
        }
#pragma unroll
      for (int i = 0; i < (DT == DT_F32 ? 2 : 1); i++) raw[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& u = raw[DT == DT_F32 ? i >> 2 : 0];
    const int k = i & 3;
    return k == 0 ? u.x : (k == 1 ? u.y : (k == 2 ? u.z : u.w));
  }
  __device__ __forceinline__ float at(int i) const {
    if (DT == DT_F32) return __uint_as_float(word(i));
    const uint32_t w = word(i >> 1);
    if (DT == DT_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    return f16_bits_to_f32((uint16_t)(i & 1 ? w >> 16 : w));
  }
  // a NaN or infinity: 0x7f800000 or more
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0;
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 8; i++) m = max(m, word(i) & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) m = __vmaxu2(m, word(i) & 0x7fff7fffu);
      m = max(m >> 16, m & 0xffffu);
      return DT == DT_BF16 ? m << 16 : __float_as_uint(f16_bits_to_f32((uint16_t)m));
    }
  }
};

// the row and first column of eight values; flat: rows lie one behind the
// other in whole groups, as the codes do
struct Spot8 {
  int64_t row, col;
};
__device__ __forceinline__ Spot8 spot8(int64_t t, int64_t groups, bool flat) {
  if (flat) return {0, t * 8};
  const int64_t g = t >> 2, row = (uint64_t)g >> 32 ? g / groups : (uint32_t)g / (uint32_t)groups;
  return {row, (g - row * groups) * kA8Group + (t & 3) * 8};
}

// Four lanes share a group, eight elements each.
template <int FMT, int DT>
__global__ void __launch_bounds__(256) act8_save_kernel(const void* x, int64_t rows, int64_t cols, int64_t ldx,
                                                        uint8_t* codes, uint8_t* scales, int wide, int flat) {
  const int64_t groups = (cols + kA8Group - 1) / kA8Group, total = rows * groups * 4;
  const int64_t t0 = (int64_t)blockIdx.x * 256 * kRuns + threadIdx.x;
  Run8<DT> v[kRuns];
#pragma unroll
  for (int r = 0; r < kRuns; r++) {
    const int64_t t = t0 + r * 256;
    const Spot8 s = spot8(t, groups, flat);
    v[r].load(x, s.row * ldx + s.col, t < total ? (flat ? 8 : (int)min((int64_t)8, cols - s.col)) : 0, wide);
  }
#pragma unroll
  for (int r = 0; r < kRuns; r++) {
    const int64_t t = t0 + r * 256;
    uint32_t amax = v[r].amax();
    const bool odd = __any_sync(0xffffffffu, amax >= 0x7f800000u);
    if (odd) {  // of the finite elements only
      amax = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t m = __float_as_uint(v[r].at(i)) & 0x7fffffffu;
        if (m < 0x7f800000u) amax = max(amax, m);
      }
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int ex = A8<FMT>::exponent(amax);
    const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
    uint32_t lo, hi;
    if (odd) {
      lo = hi = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        lo |= A8<FMT>::encode(v[r].at(i), inv) << (8 * i);
        hi |= A8<FMT>::encode(v[r].at(4 + i), inv) << (8 * i);
      }
    } else {
      lo = A8<FMT>::encode2(v[r].at(0), v[r].at(1), inv) | A8<FMT>::encode2(v[r].at(2), v[r].at(3), inv) << 16;
      hi = A8<FMT>::encode2(v[r].at(4), v[r].at(5), inv) | A8<FMT>::encode2(v[r].at(6), v[r].at(7), inv) << 16;
    }
    // eight groups of the warp: their scales in two words
    uint32_t sb = (uint32_t)(ex + 127);
    sb |= __shfl_down_sync(0xffffffffu, sb, 4) << 8;
    sb |= __shfl_down_sync(0xffffffffu, sb, 8) << 16;
    if (t >= total) continue;
    __stcs(reinterpret_cast<uint2*>(codes) + t, make_uint2(lo, hi));
    const int64_t g = t >> 2;
    if ((threadIdx.x & 15) == 0 && t + 16 <= total && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0)
      reinterpret_cast<uint32_t*>(scales)[g >> 2] = sb;
    else if ((threadIdx.x & 3) == 0 && ((t & ~(int64_t)15) + 16 > total || (reinterpret_cast<uintptr_t>(scales) & 3u)))
      scales[g] = (uint8_t)sb;
  }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(256) act8_load_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                        int64_t cols, void* out, int64_t ldo, int wide, int flat) {
  const int64_t groups = (cols + kA8Group - 1) / kA8Group, total = rows * groups * 4;
  const int64_t t0 = (int64_t)blockIdx.x * 256 * kRuns + threadIdx.x;
  uint2 c[kRuns];
  uint32_t sb[kRuns];
#pragma unroll
  for (int r = 0; r < kRuns; r++) {
    const int64_t t = min(t0 + r * 256, total - 1);
    c[r] = __ldcs(reinterpret_cast<const uint2*>(codes) + t);
    sb[r] = __ldg(scales + (t >> 2));
  }
#pragma unroll
  for (int r = 0; r < kRuns; r++) {
    const int64_t t = t0 + r * 256;
    if (t >= total) return;
    const Spot8 s = spot8(t, groups, flat);
    const int n = flat ? 8 : (int)min((int64_t)8, cols - s.col);
    if (n <= 0) continue;
    float v[8];
    a8_values8<FMT>(c[r], sb[r], v);
    if (DT == DT_F16) {
      // a finite value that rounded past float16's largest stays finite (it
      // came from a finite element); an infinity stays one
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (fabsf(v[i]) < __uint_as_float(0x7f800000u)) v[i] = fminf(fmaxf(v[i], -65504.0f), 65504.0f);
    }
    const int64_t at = s.row * ldo + s.col;
    if (wide && n == 8) {
      if (DT == DT_F32) {
        float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
        __stcs(d, make_float4(v[0], v[1], v[2], v[3]));
        __stcs(d + 1, make_float4(v[4], v[5], v[6], v[7]));
      } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++)  // bfloat16 holds the values exactly
          u[i] = DT == DT_F16 ? f32_to_f16_bits(v[2 * i]) | (uint32_t)f32_to_f16_bits(v[2 * i + 1]) << 16
                              : __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
        __stcs(reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at), make_uint4(u[0], u[1], u[2], u[3]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) store_elem(out, DT, at + i, v[i]);
    }
  }
}

static unsigned act8_grid(int64_t rows, int64_t cols) {
  return (unsigned)((rows * ((cols + kA8Group - 1) / kA8Group) * 4 + 256 * kRuns - 1) / (256 * kRuns));
}

// whether 16-byte accesses at multiples of eight columns are aligned
static int wide_rows(const void* p, int dtype, int64_t ld) {
  const int64_t e = dtype == DT_F32 ? 4 : 2;
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * e) % 16 == 0;
}

cudaError_t launch_act8_save(int fmt, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                             uint8_t* scales, cudaStream_t st) {
  const unsigned grid = act8_grid(rows, cols);
  const int w = wide_rows(x, dtype, ldx), flat = ldx == cols && cols % kA8Group == 0;
#define ODY_S(F, D) \
  if (fmt == F && dtype == D) act8_save_kernel<F, D><<<grid, 256, 0, st>>>(x, rows, cols, ldx, codes, scales, w, flat);
  ODY_S(A8_E4M3, DT_F32) ODY_S(A8_E4M3, DT_F16) ODY_S(A8_E4M3, DT_BF16)
  ODY_S(A8_E5M2, DT_F32) ODY_S(A8_E5M2, DT_F16) ODY_S(A8_E5M2, DT_BF16)
#undef ODY_S
  return cudaGetLastError();
}

cudaError_t launch_act8_load(int fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                             int dtype, int64_t ldo, cudaStream_t st) {
  const unsigned grid = act8_grid(rows, cols);
  const int w = wide_rows(out, dtype, ldo), flat = ldo == cols && cols % kA8Group == 0;
#define ODY_L(F, D) \
  if (fmt == F && dtype == D) act8_load_kernel<F, D><<<grid, 256, 0, st>>>(codes, scales, rows, cols, out, ldo, w, flat);
  ODY_L(A8_E4M3, DT_F32) ODY_L(A8_E4M3, DT_F16) ODY_L(A8_E4M3, DT_BF16)
  ODY_L(A8_E5M2, DT_F32) ODY_L(A8_E5M2, DT_F16) ODY_L(A8_E5M2, DT_BF16)
#undef ODY_L
  return cudaGetLastError();
}

}  // namespace ody
