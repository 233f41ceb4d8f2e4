// ody_linear_rows.cu -- few rows: one pass over the weight's bytes.
//
// With a handful of rows a product is bound by reading the weight, 0.5625
// (NVFP4) or 0.53125 (MXFP4) bytes an element, so its bytes go straight from
// memory through shared memory into registers, are decoded there and fed to
// mma.sync.m16n8k16 (bfloat16, float32 sums) with the weight as the 16-row
// operand and the rows as the 8 columns.  At that rate the tensor core is
// far from busy and the rows' operand fits in registers, which is why this is
// not a tcgen05 kernel: that needs both operands in shared memory.
//
// A warp works on 16 weight rows x 256 columns at a time, whatever the
// product: the forward one reduces over the columns, the input gradient over
// the rows.  The order of the reduction inside an mma is free as long as both
// operands agree, so each thread takes whole blocks:
//   forward: rows g and g + 8 of the 16 (g = lane / 4), columns 64 t to 64 t
//            + 63 (t = lane % 4); sixteen mma per 256 columns
//   dgrad:   rows 4 t to 4 t + 3, columns 32 g to 32 g + 31; neighbouring
//            rows are paired by byte permutes; sixteen mma per 16 rows
// Eight warps share the reduction, and a cluster of up to eight CTAs where
// the outputs alone do not fill the GPU; their sums are added in a fixed
// order through (distributed) shared memory.  One launch, no workspace.
//
// float16 and float32 rows are split exactly into two and three bfloat16
// parts, which take that many of the eight columns.
#include <algorithm>

#include "ody_linear_dev.cuh"
#include "ody_linear_rows.h"

namespace ody {

constexpr int kRowThreads = 256, kRowWarps = 8;
constexpr int kTileR = 16, kTileK = 256;
// A row's piece of a tile is 144 or 136 bytes at any byte offset: ten aligned
// 16-byte words.  The pitch of eleven keeps a warp's reads, eight rows by
// four offsets of nine words, on 32 different banks.
constexpr int kWords = 10, kPitch = 176;
constexpr int kTileBytes = kTileR * kPitch, kDepth = 4;
constexpr int kRowSmem = kRowWarps * kDepth * kTileBytes;

__device__ __forceinline__ uint32_t srow(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

struct RowArgs {
  LinearOut o;
  const void* a;  // x or dy
  int64_t lda;
  const uint8_t* q;
  int64_t out, in;  // weight rows and columns
  int rows;         // of a
  int wide;         // a's rows are 16-byte aligned
};

// One tile of the weight into this warp's stage: rows r0.., columns k0.. (of
// kTileK).  Words that lie wholly inside the weight's bytes are copied
// asynchronously, the first and last bytes of the weight one by one.
template <int KIND>
__device__ __forceinline__ void fetch_tile(const RowArgs& a, uint8_t* st, int64_t r0, int64_t k0, int lane) {
  using W = W4<KIND>;
  const int64_t per = a.in / W::BE;  // blocks in a row
  const uint8_t* end = a.q + a.out * per * W::SB;
#pragma unroll
  for (int i = 0; i < kTileR * kWords / 32; i++) {
    const int c = i * 32 + lane, r = c / kWords, w = c - r * kWords;
    if (r0 + r < a.out) {
      const uint8_t* src = a.q + ((r0 + r) * per + k0 / W::BE) * W::SB;
      const uint8_t* p = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15) + w * 16;
      uint8_t* d = st + r * kPitch + w * 16;
      if (p >= a.q && p + 16 <= end) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(srow(d)), "l"(p) : "memory");
      } else if (p < end && p + 16 > a.q) {
        for (int b = 0; b < 16; b++)
          if (p + b >= a.q && p + b < end) d[b] = p[b];
      }
    }
  }
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}

// Eight weights as bfloat16 pairs, from a word of four code bytes: o[i] holds
// nibbles i and i + 4, that is weights {1, 5}, {0, 4}, {3, 7}, {2, 6}, times
// 2^-126 (see w4_raw8).
template <int KIND>
__device__ __forceinline__ void raw_pairs(uint32_t w, uint32_t o[4]) {
  if (KIND != Q_MXFP4_OCP) w &= ~0x11111111u | (w >> 1) | (w >> 2);
  o[0] = ((w << 12) & 0x80008000u) | ((w << 6) & 0x01c001c0u);
  o[1] = ((w << 8) & 0x80008000u) | ((w << 2) & 0x01c001c0u);
  o[2] = ((w << 4) & 0x80008000u) | ((w >> 2) & 0x01c001c0u);
  o[3] = (w & 0x80008000u) | ((w >> 6) & 0x01c001c0u);
}

// 2^kBias times less than the weight is what the mma sees: NVFP4's scales
// then fit one bfloat16 factor together with 2^126
template <int KIND>
struct Bias {
  static constexpr int value = W4<KIND>::MX ? 0 : 9;
};
// The factors that bring raw pairs to weights * 2^-kBias: one, or where a
// power of two above 2 makes 2^126 * scale overflow, two.
template <int KIND>
__device__ __forceinline__ uint32_t one_factor(uint32_t byte) {
  if (KIND == Q_MXFP4 || KIND == Q_MXFP4_OCP) {
    const uint32_t h = (KIND == Q_MXFP4 && byte == 0) ? 0u : (byte + 126) << 7;
    return h | h << 16;
  }
  // E4M3 as float16, exact; times 2^117
  const uint32_t h = __float_as_uint(__fmul_rn(e4m3_to_f32((uint8_t)byte), 1.661534994731145e35f)) >> 16;
  return h | h << 16;
}

// NW code words of a block and its scale byte
template <int NW>
__device__ __forceinline__ void load_block(const uint8_t* p, uint32_t w[NW], uint32_t& scale) {
  const uint32_t sh = 8 * ((uint32_t)reinterpret_cast<uintptr_t>(p) & 3);
  const uint32_t* s = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
  uint32_t v[NW + 1];
#pragma unroll
  for (int i = 0; i <= NW; i++) v[i] = s[i];
#pragma unroll
  for (int i = 0; i < NW; i++) w[i] = __funnelshift_r(v[i], v[i + 1], sh);
  scale = (v[NW] >> sh) & 0xffu;  // the byte behind the codes
}

__device__ __forceinline__ void mma16816(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int DT>
__device__ __forceinline__ uint16_t part_of(float v, int part) {
  uint16_t h[3];
  split_bf16(v, h[0], h[1], h[2]);
  return part == 0 ? h[0] : (part == 1 ? h[1] : h[2]);
}

// N consecutive elements of a row (from column k, zeros behind `cols`), this
// lane's part of them, packed in pairs
template <int DT, int N>
__device__ __forceinline__ void load_rows(const void* row, int64_t k, int64_t cols, int wide, int part, uint32_t o[N / 2]) {
  if (wide && k + N <= cols) {
    if (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < N / 4; i++) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k) + i);
        o[2 * i] = part_of<DT>(f.x, part) | (uint32_t)part_of<DT>(f.y, part) << 16;
        o[2 * i + 1] = part_of<DT>(f.z, part) | (uint32_t)part_of<DT>(f.w, part) << 16;
      }
    } else {
      if (N == 4) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(row) + k));
        o[0] = u.x, o[1] = u.y;
      }
#pragma unroll
      for (int i = 0; i < N / 8; i++) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(row) + k) + i);
        o[4 * i] = u.x, o[4 * i + 1] = u.y, o[4 * i + 2] = u.z, o[4 * i + 3] = u.w;
      }
      if (DT == DT_F16) {
#pragma unroll
        for (int i = 0; i < N / 2; i++)
          o[i] = part_of<DT>(f16_bits_to_f32(o[i] & 0xffff), part) |
                 (uint32_t)part_of<DT>(f16_bits_to_f32(o[i] >> 16), part) << 16;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      uint32_t h[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int64_t c = k + 2 * i + j;
        if (DT == DT_BF16)
          h[j] = c < cols ? reinterpret_cast<const uint16_t*>(row)[c] : 0u;
        else
          h[j] = c < cols ? part_of<DT>(load_elem(row, DT, c), part) : 0u;
      }
      o[i] = h[0] | h[1] << 16;
    }
  }
}

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

// Adds what `n` floats of every warp (at red + warp * n) and every CTA of the
// cluster hold, always in the same order, and stores `count` results: result
// o is the sum of the `parts` sums at place(o), place(o) + step, ...
template <class Place, class Store>
__device__ __forceinline__ void add_and_store(float* red, int n, int count, int parts, int step, Place&& place,
                                              Store&& store) {
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kRowThreads) {
    float v = red[i];
#pragma unroll
    for (int w = 1; w < kRowWarps; w++) v = __fadd_rn(v, red[w * n + i]);
    red[i] = v;
  }
  if (ranks > 1)
    cluster_barrier();
  else
    __syncthreads();
  for (int o = rank * kRowThreads + threadIdx.x; o < count; o += ranks * kRowThreads) {
    const int at = place(o);
    float sum = 0.0f;
    for (int p = 0; p < parts; p++) {
      float v = ranks > 1 ? peer_float(red + at + p * step, 0) : red[at + p * step];
      for (uint32_t r = 1; r < ranks; r++) v = __fadd_rn(v, peer_float(red + at + p * step, r));
      sum = p ? __fadd_rn(sum, v) : v;
    }
    store(o, sum);
  }
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

// where this lane's columns of the mma come from: row c / parts of a, its part c % parts
template <int DT, int NT>
struct Columns {
  const uint8_t* row[NT];
  int part[NT];
  __device__ __forceinline__ Columns(const RowArgs& a, int g) {
    constexpr int P = bf16_parts(DT), ES = DT == DT_F32 ? 4 : 2;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int c = n * 8 + g, m = c / P;
      part[n] = c - m * P;
      row[n] = m < a.rows ? reinterpret_cast<const uint8_t*>(a.a) + (int64_t)m * a.lda * ES : nullptr;
    }
  }
};

// the steps of one warp and its ring of stages
struct Walk {
  uint8_t* ring;
  int64_t me, stride;
  int slot = 0;
  __device__ __forceinline__ Walk(uint8_t* sm, int warp) {
    ring = sm + warp * kDepth * kTileBytes;
    stride = (int64_t)kRowWarps * cluster_size();
    me = (int64_t)cluster_rank() * kRowWarps + warp;
  }
  template <int KIND, class At>
  __device__ __forceinline__ void start(const RowArgs& a, int64_t steps, At&& at, int lane) {
#pragma unroll
    for (int i = 0; i < kDepth - 1; i++) {
      const int64_t s = me + i * stride;
      if (s < steps) fetch_tile<KIND>(a, ring + i * kTileBytes, at(s).r, at(s).k, lane);
      fetch_commit();
    }
  }
  // the stage of step s, once it is there; the step kDepth - 1 after it is asked for
  template <int KIND, class At>
  __device__ __forceinline__ const uint8_t* next(const RowArgs& a, int64_t s, int64_t steps, At&& at, int lane) {
    const int64_t nx = s + (kDepth - 1) * stride;
    __syncwarp();
    if (nx < steps) fetch_tile<KIND>(a, ring + ((slot + kDepth - 1) & (kDepth - 1)) * kTileBytes, at(nx).r, at(nx).k, lane);
    fetch_commit();
    fetch_wait<kDepth - 1>();
    const uint8_t* st = ring + slot * kTileBytes;
    slot = (slot + 1) & (kDepth - 1);
    return st;
  }
};
struct Spot {
  int64_t r, k;
};

// byte offset of (row, column) of the weight inside its aligned 16-byte word
template <int KIND>
__device__ __forceinline__ int skew(const RowArgs& a, int64_t r, int64_t k) {
  using W = W4<KIND>;
  return (int)((reinterpret_cast<uintptr_t>(a.q) + (uint64_t)(r * (a.in / W::BE) + k / W::BE) * W::SB) & 15);
}

// NR rows' raw pairs of one code word, brought to weights
template <int KIND, int NR>
__device__ __forceinline__ void scaled_pairs(const uint32_t w[NR], const uint32_t s[NR], const uint32_t f[NR], bool two,
                                             uint32_t o[NR][4]) {
#pragma unroll
  for (int r = 0; r < NR; r++) {
    raw_pairs<KIND>(w[r], o[r]);
#pragma unroll
    for (int j = 0; j < 4; j++) o[r][j] = mul_bf16x2(o[r][j], f[r]);
  }
  if (W4<KIND>::MX && two) {
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const uint32_t h = w4_scale_bf16x2<KIND>(s[r]);
#pragma unroll
      for (int j = 0; j < 4; j++) o[r][j] = mul_bf16x2(o[r][j], h);
    }
  }
}
// whether any lane's power of two is too large for one factor
template <int KIND, int NR>
__device__ __forceinline__ bool factors(const uint32_t s[NR], uint32_t f[NR]) {
  bool two = false;
  if (W4<KIND>::MX) {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < NR; r++) m = max(m, s[r]);
    two = __any_sync(0xffffffffu, m > 128u);
  }
#pragma unroll
  for (int r = 0; r < NR; r++) f[r] = two ? kTwo126 : one_factor<KIND>(s[r]);
  return two;
}

// y[m, n] for 16 weight rows n per cluster; NT * 8 columns of the mma hold
// rows x parts
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_forward_kernel(const RowArgs a) {
  using W = W4<KIND>;
  constexpr int P = bf16_parts(DT), NWB = W::BE / 8, BLOCKS = 64 / W::BE, C = NT * 8;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t r0 = (int64_t)(blockIdx.x / cluster_size()) * kTileR;
  const int64_t steps = (a.in + kTileK - 1) / kTileK;
  const auto at = [&](int64_t s) { return Spot{r0, s * kTileK}; };
  const Columns<DT, NT> cols(a, g);
  float acc[NT][4] = {};
  Walk walk(sm, warp);
  walk.start<KIND>(a, steps, at, lane);
#pragma unroll 1
  for (int64_t s = walk.me; s < steps; s += walk.stride) {
    const int64_t k0 = s * kTileK + 64 * t;
    // few columns: this lane's 64 elements of its rows come while the weight does
    uint32_t x[NT <= 2 ? NT : 1][32];
    if (NT <= 2) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int i = 0; i < 32; i++) x[n][i] = 0;
        if (cols.row[n])
#pragma unroll
          for (int b = 0; b < 4; b++) load_rows<DT, 16>(cols.row[n], k0 + 16 * b, a.in, a.wide, cols.part[n], x[n] + 8 * b);
      }
    }
    const uint8_t* st = walk.next<KIND>(a, s, steps, at, lane);
    const uint8_t* p[2] = {st + g * kPitch + skew<KIND>(a, r0 + g, s * kTileK) + t * BLOCKS * W::SB,
                           st + (g + 8) * kPitch + skew<KIND>(a, r0 + g + 8, s * kTileK) + t * BLOCKS * W::SB};
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
      const int64_t k = k0 + b * W::BE;
      uint32_t w[2][NWB], sc[2], f[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        load_block<NWB>(p[r] + b * W::SB, w[r], sc[r]);
        if (k >= a.in) {  // behind the row's end lie other rows' bytes, or none
          sc[r] = 56;
#pragma unroll
          for (int i = 0; i < NWB; i++) w[r][i] = 0;
        }
      }
      const bool two = factors<KIND, 2>(sc, f);
#pragma unroll
      for (int i = 0; i < NWB; i++) {
        const uint32_t ww[2] = {w[0][i], w[1][i]};
        uint32_t o[2][4];
        scaled_pairs<KIND, 2>(ww, sc, f, two, o);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          uint32_t v[4];
          if (NT <= 2) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = x[NT <= 2 ? n : 0][(b * NWB + i) * 4 + j];
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = 0;
            if (cols.row[n]) load_rows<DT, 8>(cols.row[n], k + i * 8, a.in, a.wide, cols.part[n], v);
          }
          // the pairs' order: {1, 5}, {0, 4}, {3, 7}, {2, 6}
          mma16816(acc[n], o[0][0], o[1][0], o[0][1], o[1][1], __byte_perm(v[0], v[2], 0x7632),
                   __byte_perm(v[0], v[2], 0x5410));
          mma16816(acc[n], o[0][2], o[1][2], o[0][3], o[1][3], __byte_perm(v[1], v[3], 0x7632),
                   __byte_perm(v[1], v[3], 0x5410));
        }
      }
    }
  }
  fetch_wait<0>();
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);  // [warp][weight row][column]
#pragma unroll
  for (int n = 0; n < NT; n++) {
    float* d = red + warp * kTileR * C + n * 8 + 2 * t;
    d[g * C] = acc[n][0], d[g * C + 1] = acc[n][1];
    d[(g + 8) * C] = acc[n][2], d[(g + 8) * C + 1] = acc[n][3];
  }
  const float scale = __fmul_rn(out_scale(a.o), (float)(1 << Bias<KIND>::value));
  add_and_store(
      red, kTileR * C, kTileR * a.rows, P, 1, [&](int o) { return (o & 15) * C + (o >> 4) * P; },
      [&](int o, float v) {
        if (r0 + (o & 15) < a.out) finish(a.o, scale, o >> 4, r0 + (o & 15), v);
      });
}

// dx[m, k] for 256 columns k per cluster
constexpr int kRedPitch = kTileK + 8;  // a column's sums: 33 floats per 32 k, so that the eight g's differ in bank
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, NT == 1 ? 2 : 1) rows_dgrad_kernel(const RowArgs a) {
  using W = W4<KIND>;
  constexpr int P = bf16_parts(DT), NWB = W::BE / 8, BLOCKS = 32 / W::BE, C = NT * 8;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t k0 = (int64_t)(blockIdx.x / cluster_size()) * kTileK;
  const int64_t steps = (a.out + kTileR - 1) / kTileR;
  const auto at = [&](int64_t s) { return Spot{s * kTileR, k0}; };
  const Columns<DT, NT> cols(a, g);
  float acc[16][NT][4] = {};
  Walk walk(sm, warp);
  walk.start<KIND>(a, steps, at, lane);
#pragma unroll 1
  for (int64_t s = walk.me; s < steps; s += walk.stride) {
    const int64_t n0 = s * kTileR + 4 * t;
    uint32_t y[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      y[n][0] = y[n][1] = 0;
      if (cols.row[n]) load_rows<DT, 4>(cols.row[n], n0, a.out, a.wide, cols.part[n], y[n]);
    }
    const uint8_t* st = walk.next<KIND>(a, s, steps, at, lane);
    const uint8_t* p[4];
#pragma unroll
    for (int r = 0; r < 4; r++)
      p[r] = st + (4 * t + r) * kPitch + skew<KIND>(a, n0 + r, k0) + g * BLOCKS * W::SB;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
      uint32_t w[4][NWB], sc[4], f[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        load_block<NWB>(p[r] + b * W::SB, w[r], sc[r]);
        if (n0 + r >= a.out) {  // behind the last row: whatever the stage held
          sc[r] = 56;
#pragma unroll
          for (int i = 0; i < NWB; i++) w[r][i] = 0;
        }
      }
      const bool two = factors<KIND, 4>(sc, f);
#pragma unroll
      for (int i = 0; i < NWB; i++) {
        const uint32_t ww[4] = {w[0][i], w[1][i], w[2][i], w[3][i]};
        uint32_t o[4][4];
        scaled_pairs<KIND, 4>(ww, sc, f, two, o);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int n = 0; n < NT; n++)
            mma16816(acc[(b * NWB + i) * 4 + j][n], __byte_perm(o[0][j], o[1][j], 0x5410),
                     __byte_perm(o[0][j], o[1][j], 0x7632), __byte_perm(o[2][j], o[3][j], 0x5410),
                     __byte_perm(o[2][j], o[3][j], 0x7632), y[n][0], y[n][1]);
      }
    }
  }
  fetch_wait<0>();
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);  // [warp][column][33 floats per 32 k]
#pragma unroll
  for (int q = 0; q < 16; q++) {
    // the pair's two weights: {1, 5}, {0, 4}, {3, 7}, {2, 6} of word q / 4
    constexpr int first[4] = {1, 0, 3, 2};
    const int e = (q >> 2) * 8 + first[q & 3];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float* d = red + (warp * C + n * 8 + 2 * t) * kRedPitch + 33 * g + e;
      d[0] = acc[q][n][0], d[kRedPitch] = acc[q][n][1];
      d[4] = acc[q][n][2], d[kRedPitch + 4] = acc[q][n][3];
    }
  }
  const float scale = __fmul_rn(out_scale(a.o), (float)(1 << Bias<KIND>::value));
  add_and_store(
      red, C * kRedPitch, kTileK * a.rows, P, kRedPitch,
      [&](int o) { return (o >> 8) * P * kRedPitch + 33 * ((o & 255) >> 5) + (o & 31); },
      [&](int o, float v) {
        if (k0 + (o & 255) < a.in) finish(a.o, scale, o >> 8, k0 + (o & 255), v);
      });
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

template <class K>
cudaError_t launch_rows(K kernel, const RowArgs& a, int64_t tiles, int64_t steps, int smem, int sms, cudaStream_t st) {
  // enough CTAs for two per SM if there are steps for their warps
  int cluster = 1;
  while (cluster < 8 && tiles * cluster * 2 <= 2 * sms && (int64_t)cluster * kRowWarps < steps) cluster *= 2;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * cluster));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int KIND, int DT, int NT>
cudaError_t launch_one(const LinearArgs& l, const RowArgs& a, int sms, cudaStream_t st) {
  if (l.op == LIN_FORWARD)
    return launch_rows(rows_forward_kernel<KIND, DT, NT>, a, (a.out + kTileR - 1) / kTileR, (a.in + kTileK - 1) / kTileK,
                       kRowSmem, sms, st);
  if constexpr (NT <= 2) {
    constexpr int red = kRowWarps * NT * 8 * kRedPitch * 4;
    return launch_rows(rows_dgrad_kernel<KIND, DT, NT>, a, (a.in + kTileK - 1) / kTileK, (a.out + kTileR - 1) / kTileR,
                       red > kRowSmem ? red : kRowSmem, sms, st);
  }
  return cudaErrorInvalidValue;
}

template <int KIND, int DT>
cudaError_t launch_nt(const LinearArgs& l, const RowArgs& a, int sms, cudaStream_t st) {
  const int columns = a.rows * bf16_parts(DT);
  if (columns <= 8) return launch_one<KIND, DT, 1>(l, a, sms, st);
  if (columns <= 16) return launch_one<KIND, DT, 2>(l, a, sms, st);
  return launch_one<KIND, DT, 4>(l, a, sms, st);
}

template <int KIND>
cudaError_t launch_dt(const LinearArgs& l, const RowArgs& a, int sms, cudaStream_t st) {
  if (l.a_dtype == DT_F32) return launch_nt<KIND, DT_F32>(l, a, sms, st);
  if (l.a_dtype == DT_F16) return launch_nt<KIND, DT_F16>(l, a, sms, st);
  return launch_nt<KIND, DT_BF16>(l, a, sms, st);
}

}  // namespace

bool few_rows(const LinearArgs& a) {
  if (a.op == LIN_WGRAD) return false;
  const int be = a.kind == Q_MXFP4 || a.kind == Q_MXFP4_OCP ? 32 : 16;
  return a.in % be == 0 && a.rows * bf16_parts(a.a_dtype) <= (a.op == LIN_FORWARD ? 32 : 16);
}

cudaError_t launch_few_rows(const LinearArgs& l, int sms, cudaStream_t st) {
  RowArgs a;
  a.o = l.o;
  a.a = l.a, a.lda = l.lda;
  a.q = l.q;
  a.out = l.out, a.in = l.in;
  a.rows = (int)l.rows;
  a.wide = (reinterpret_cast<uintptr_t>(l.a) & 15u) == 0 && (l.lda * (l.a_dtype == DT_F32 ? 4 : 2)) % 16 == 0;
  if (l.kind == Q_MXFP4) return launch_dt<Q_MXFP4>(l, a, sms, st);
  if (l.kind == Q_MXFP4_OCP) return launch_dt<Q_MXFP4_OCP>(l, a, sms, st);
  return launch_dt<Q_NVFP4>(l, a, sms, st);
}

}  // namespace ody
