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
// Products on the FP32 pipe: 64 x 64 tiles, 256 threads with 4 x 4 results
// each, 16 steps of the reduction at a time through shared memory.  Sums run
// in float32, in two levels (64 products, then their sums), so that rounding
// errors grow with the root of the number of partial sums only.
// ---------------------------------------------------------------------------
constexpr int kFT = 64, kFK = 16;

template <int OP, int KIND>
__global__ void __launch_bounds__(256) linear_fp32_kernel(LinearArgs p) {
  __shared__ float As[kFK][kFT + 4], Bs[kFK][kFT + 4];
  const int64_t M = OP == LIN_WGRAD ? p.out : p.rows, N = OP == LIN_FORWARD ? p.out : p.in;
  const int64_t R = OP == LIN_FORWARD ? p.in : (OP == LIN_DGRAD ? p.out : p.rows);
  const int64_t tn = (N + kFT - 1) / kFT;
  const int64_t m0 = ((int64_t)blockIdx.x / tn) * kFT, n0 = ((int64_t)blockIdx.x % tn) * kFT;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t groups = (p.in + kA8Group - 1) / kA8Group;
  float acc[4][4] = {}, part[4][4] = {};
  for (int64_t r0 = 0; r0 < R; r0 += kFK) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int t = threadIdx.x + 256 * i;
      // the index that is contiguous in memory runs fastest over the threads
      const int ar = OP == LIN_WGRAD ? t / kFT : t % kFK, am = OP == LIN_WGRAD ? t % kFT : t / kFK;
      const int64_t m = m0 + am, ra = r0 + ar;
      float v = 0.0f;
      if (m < M && ra < R) v = load_elem(p.a, p.a_dtype, OP == LIN_WGRAD ? ra * p.lda + m : m * p.lda + ra);
      As[ar][am] = v;
      const int br = OP == LIN_FORWARD ? t % kFK : t / kFT, bn = OP == LIN_FORWARD ? t / kFK : t % kFT;
      const int64_t n = n0 + bn, rb = r0 + br;
      v = 0.0f;
      if (n < N && rb < R) {
        if constexpr (OP == LIN_WGRAD)
          v = a8_value<KIND>(p.q[(rb * groups) * kA8Group + n], p.scales[rb * groups + n / kA8Group]);
        else
          v = W4<KIND>::at(p.q, OP == LIN_FORWARD ? n * p.in + rb : rb * p.in + n);
      }
      Bs[br][bn] = v;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kFK; k++) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = As[k][ty * 4 + i], b[i] = Bs[k][tx + 16 * i];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) part[i][j] = __fmaf_rn(a[i], b[j], part[i][j]);
    }
    __syncthreads();
    if ((r0 / kFK) % 4 == 3 || r0 + kFK >= R) {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __fadd_rn(acc[i][j], part[i][j]), part[i][j] = 0.0f;
    }
  }
  const float s = out_scale(p.o);
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m < M && n < N) finish(p.o, s, m, n, acc[i][j]);
    }
}

template <int OP, int KIND>
static cudaError_t launch_fp32(const LinearArgs& a, cudaStream_t st) {
  const int64_t M = OP == LIN_WGRAD ? a.out : a.rows, N = OP == LIN_FORWARD ? a.out : a.in;
  const int64_t tiles = ((M + kFT - 1) / kFT) * ((N + kFT - 1) / kFT);
  linear_fp32_kernel<OP, KIND><<<(unsigned)tiles, 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <int OP>
static cudaError_t launch_fp32_w4(const LinearArgs& a, cudaStream_t st) {
  switch (a.kind) {
    case Q_MXFP4:
      return launch_fp32<OP, Q_MXFP4>(a, st);
    case Q_MXFP4_OCP:
      return launch_fp32<OP, Q_MXFP4_OCP>(a, st);
    default:  // the tensor scale of ODY_Q_NVFP4_TENSOR is applied to the sums
      return launch_fp32<OP, Q_NVFP4>(a, st);
  }
}

static int lin_sms() {
  static int n[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (!n[dev]) cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
  return n[dev] ? n[dev] : 148;
}

// Few products are done by the FP32 pipe in one launch; more go to the tensor
// cores, after their operands have been brought to bfloat16.
static bool small_product(const LinearArgs& a) { return (double)a.rows * a.out * a.in <= 0; }

// (of any kind: the query does not name one, so widths are taken to be in 32s)
int64_t linear_workspace(const LinearArgs& a) {
  return small_product(a) || (few_rows(a) && a.in % 32 == 0) ? 0 : gemm_workspace(a, lin_sms());
}

cudaError_t launch_linear(const LinearArgs& a, void* ws, cudaStream_t st) {
  if (few_rows(a)) return launch_few_rows(a, lin_sms(), st);
  if (!small_product(a)) return launch_gemm(a, ws, lin_sms(), st);
  if (a.op == LIN_FORWARD) return launch_fp32_w4<LIN_FORWARD>(a, st);
  if (a.op == LIN_DGRAD) return launch_fp32_w4<LIN_DGRAD>(a, st);
  return a.kind == A8_E4M3 ? launch_fp32<LIN_WGRAD, A8_E4M3>(a, st) : launch_fp32<LIN_WGRAD, A8_E5M2>(a, st);
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
