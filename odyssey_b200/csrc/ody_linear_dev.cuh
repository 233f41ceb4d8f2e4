// ody_linear_dev.cuh -- device pieces shared by the quantised linear layer's
// kernels: decoding of 4-bit weights and 8-bit activations, element access,
// the last step of a result.
#pragma once
#include "ody_linear.h"
#include "ody_numerics.cuh"

namespace ody {

template <int KIND>
struct W4 {
  static constexpr bool MX = KIND == Q_MXFP4 || KIND == Q_MXFP4_OCP;
  static constexpr int BE = MX ? 32 : 16;  // elements per block
  static constexpr int SB = MX ? 17 : 9;   // bytes per block
};

// ---- eight weights at once, as bfloat16 pairs -------------------------------
// Code times scale is exact in bfloat16 for finite scales: two bits of value
// times at most four of scale.  Code 1 is 0.5 in the OCP kind and 0 in the
// others.
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// a block's scale as a bfloat16 pair (exact): E8M0 (in the OCP kind 0 is
// 2^-127 and 255 NaN) or E4M3
template <int KIND>
__device__ __forceinline__ uint32_t w4_scale_bf16x2(uint32_t byte) {
  uint32_t h;
  if (KIND == Q_MXFP4)
    h = byte << 7;  // 0 is 0, 255 is infinity
  else if (KIND == Q_MXFP4_OCP)
    h = byte == 0xFF ? 0x7fc0u : (byte ? byte << 7 : 0x0040u);
  else
    h = __float_as_uint(e4m3_to_f32((uint8_t)byte)) >> 16;
  return h | h << 16;
}
// Four code bytes (eight weights, the first in the lowest byte's high nibble)
// as o[i] = weights 2i, 2i + 1, times 2^-126: the code's three magnitude bits
// put where bfloat16 keeps the lowest two exponent bits and the highest
// mantissa bit (0.5 as a subnormal), its sign on top.  Only the OCP kind has
// 0.5; in the others that code is zero.
template <int KIND>
__device__ __forceinline__ void w4_raw8(uint32_t w, uint32_t o[4]) {
  if (KIND != Q_MXFP4_OCP) w &= ~0x11111111u | (w >> 1) | (w >> 2);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    // byte i: its high nibble to bits 12..15, its low one to bits 28..31
    const uint32_t t = ((w >> (8 * i)) & 0xffu) * 0x10000100u;
    o[i] = (t & 0x80008000u) | ((t >> 6) & 0x01c001c0u);
  }
}
constexpr uint32_t kTwo126 = 0x7e807e80u;  // 2^126 as a bfloat16 pair

// the values of eight codes
template <int FMT>
__device__ __forceinline__ void a8_values8(uint2 c, uint32_t scale_byte, float v[8]) {
  const float f = __uint_as_float(scale_byte << 23);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t two = (i < 2 ? c.x : c.y) >> (16 * (i & 1));
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, FMT == A8_E4M3 ? __NV_E4M3 : __NV_E5M2);
    v[2 * i] = __fmul_rn(f16_bits_to_f32(h.x), f), v[2 * i + 1] = __fmul_rn(f16_bits_to_f32(h.y), f);
  }
}

// Eight neighbouring elements of the quantised operand: codes in their order
// (weight i in nibble i ^ 1), scales, and as bfloat16.  Weights of rows that
// are not a multiple of eight wide may begin at any nibble and reach into a
// second block.
template <int OP, int KIND>
struct EightQ {
  uint32_t code[OP == LIN_WGRAD ? 2 : 1], scale;  // scale: of the elements before `split`, and 8 bits up the others'
  int split;
  // row r, column c; n elements are there (8 where blocks)
  __device__ __forceinline__ void load(const uint8_t* q, const uint8_t* scales, int64_t in, int64_t r, int64_t c, int n,
                                       bool blocks) {
    split = 8;
    if constexpr (OP == LIN_WGRAD) {
      const int64_t groups = (in + kA8Group - 1) / kA8Group;
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(q + r * groups * kA8Group + c));
      code[0] = u.x, code[1] = u.y;
      scale = __ldg(scales + r * groups + c / kA8Group);
    } else {
      using W = W4<KIND>;
      const uint64_t e = (uint64_t)(r * in + c);
      const uint8_t* const blk = q + e / W::BE * W::SB;
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
      float v[8];
      a8_values8<KIND>(make_uint2(code[0], code[1]), scale, v);
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
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

__device__ __forceinline__ float load_elem(const void* p, int dt, int64_t i) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == DT_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
}
__device__ __forceinline__ void store_elem(void* p, int dt, int64_t i, float v) {
  if (dt == DT_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<uint16_t*>(p)[i] = dt == DT_F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v);
}

__device__ __forceinline__ float out_scale(const LinearOut& o) {
  return o.tscale ? __fmul_rn(o.alpha, *o.tscale) : o.alpha;
}
__device__ __forceinline__ void finish(const LinearOut& o, float s, int64_t i, int64_t j, float acc) {
  const int64_t at = i * o.ld + j;
  float v = __fmul_rn(acc, s);
  if (o.add) v = __fadd_rn(v, load_elem(o.add, o.dtype, at));
  store_elem(o.c, o.dtype, at, v);
}

// A float32 as the exact sum of three bfloat16 (float16: of two): each part
// is the rest cut to bfloat16's eight bits, so no part is ever larger than
// the value (rounding up could pass the largest finite one).  A non-finite
// value is its first part alone, since inf - inf would spoil the others.
__device__ __forceinline__ void split_bf16(float x, uint16_t& a, uint16_t& b, uint16_t& c) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    a = (u & 0x7fffffu) ? 0x7fc0 : (uint16_t)(u >> 16);
    b = c = 0;
    return;
  }
  a = (uint16_t)(u >> 16);
  const float r = __fsub_rn(x, __uint_as_float(u & 0xffff0000u));
  const uint32_t v = __float_as_uint(r);
  b = (uint16_t)(v >> 16);
  c = (uint16_t)(__float_as_uint(__fsub_rn(r, __uint_as_float(v & 0xffff0000u))) >> 16);
}
// parts an element of this type takes
__host__ __device__ constexpr int bf16_parts(int dtype) { return dtype == DT_F32 ? 3 : (dtype == DT_F16 ? 2 : 1); }

__device__ __forceinline__ void mma16816(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- clusters ---------------------------------------------------------------
__device__ __forceinline__ uint32_t srow(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(srow(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace ody
