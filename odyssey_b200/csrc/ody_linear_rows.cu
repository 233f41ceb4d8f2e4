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
// A warp works on 16 weight rows x 256 columns (forward) or 128 columns
// (dgrad) at a time.  The order of the reduction inside an mma is free as
// long as both operands agree, so each thread takes runs of 16 weights:
//   forward: rows g and g + 8 of the 16 (g = lane / 4), columns 64 t to 64 t
//            + 63 (t = lane % 4), four runs; the reduction is over columns
//   dgrad:   rows 4 t to 4 t + 3, columns 16 g to 16 g + 15; the reduction is
//            over rows, so neighbouring rows are paired by byte permutes
// Forward, eight warps take 128 weight rows and the same columns, so that the
// CTA's threads bring x's piece in once, already cut into bfloat16 parts, for
// all of them; dgrad, eight warps share the reduction over the rows.  In both
// a cluster of up to eight CTAs shares it too where the outputs alone do not
// fill the GPU.  Sums are added in a fixed order through (distributed) shared
// memory.  One launch, no workspace.
//
// The loops are kept rolled and what they do exists once: a launch of a few
// microseconds reads its code cold, and with everything unrolled (16 KB) that
// took longer than the weight.
//
// float16 and float32 rows are split exactly into two and three bfloat16
// parts, which take that many of the eight columns.
#include <algorithm>

#include "ody_linear_dev.cuh"
#include "ody_linear_rows.h"

namespace ody {

constexpr int kRowThreads = 256, kRowWarps = 8, kTileR = 16, kDepth = 4;  // kDepth: dgrad's stages

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

// A warp's ring of weight tiles, 16 rows x K columns each.  A row's piece is
// at most K * 9 / 16 bytes at any byte offset, so it is copied as the aligned
// 16-byte words around it.  For 256 columns the pitch of eleven words keeps a
// warp's reads, eight rows by four offsets of nine words, on 32 banks.
template <int KIND, int K>
struct Ring {
  using W = W4<KIND>;
  static constexpr int WORDS = (K * 9 / 16 + 30) / 16, PITCH = (WORDS | 1) * 16, BYTES = kTileR * PITCH;
  static constexpr int COPIES = kTileR * WORDS / 32;
  static_assert(kTileR * WORDS % 32 == 0 && K % 128 == 0, "whole copies per lane");

  // Columns k0.. of rows r0.. into a stage.  Words that lie wholly inside the
  // weight's bytes are copied asynchronously; the first and the last bytes of
  // the weight one by one.
  static __device__ __forceinline__ void fetch(const RowArgs& a, uint8_t* st, int64_t r0, int64_t k0, int lane) {
    const int64_t row_bytes = a.in / W::BE * W::SB;
    const uint8_t* const end = a.q + a.out * row_bytes;
    const uint8_t* const first = a.q + r0 * row_bytes + k0 / W::BE * W::SB;
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
      const int c = i * 32 + lane, r = c / WORDS, w = c - r * WORDS;
      if (r0 + r >= a.out) continue;
      const uint8_t* p =
          reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(first + r * row_bytes) & ~(uintptr_t)15) + w * 16;
      uint8_t* d = st + r * PITCH + w * 16;
      if (p >= a.q && p + 16 <= end) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(srow(d)), "l"(p) : "memory");
      } else {
#pragma unroll 1
        for (int b = 0; b < 16; b++)
          if (p + b >= a.q && p + b < end) d[b] = p[b];
      }
    }
  }
  // where (row r, column k) of the weight, at column c of the tile's row, lies in a stage
  static __device__ __forceinline__ int place(const RowArgs& a, int64_t r, int64_t k0, int tile_row) {
    const uint64_t at = reinterpret_cast<uintptr_t>(a.q) + (uint64_t)(r * (a.in / W::BE) + k0 / W::BE) * W::SB;
    return tile_row * PITCH + (int)(at & 15);
  }
};

// Sixteen weights from column c (a multiple of 16) of a row whose first block
// is at p: two words of codes and the block's scale byte.
template <int KIND>
__device__ __forceinline__ void load_run(const uint8_t* p, int c, uint32_t w[2], uint32_t& scale) {
  using W = W4<KIND>;
  p += c / W::BE * W::SB;
  const uint8_t* q = p + c % W::BE / 2;
  const uint32_t sh = 8 * ((uint32_t)reinterpret_cast<uintptr_t>(q) & 3);
  const uint32_t* s = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(q) & ~(uintptr_t)3);
  const uint32_t v0 = s[0], v1 = s[1], v2 = s[2];
  w[0] = __funnelshift_r(v0, v1, sh);
  w[1] = __funnelshift_r(v1, v2, sh);
  scale = W::MX ? p[16] : (v2 >> sh) & 0xffu;
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

// The mma sees NVFP4 weights times 2^-9: 2^126 and every E4M3 scale then fit
// one bfloat16 factor.  A power of two above 2 does not fit one with 2^126:
// where a lane has one (weights of 8 and more), two factors are used.
template <int KIND>
__device__ __forceinline__ uint32_t one_factor(uint32_t byte) {
  if (W4<KIND>::MX) {
    const uint32_t h = (KIND == Q_MXFP4 && byte == 0) ? 0u : (byte + 126) << 7;
    return h | h << 16;
  }
  // E4M3 as float16, exact; times 2^117
  return __byte_perm(__float_as_uint(__fmul_rn(e4m3_to_f32((uint8_t)byte), 1.661534994731145e35f)), 0, 0x3232);
}
template <int KIND>
__device__ __forceinline__ float bias() {
  return W4<KIND>::MX ? 1.0f : 512.0f;
}

// NR rows' runs of 16 weights as pairs: o[row][word][pair]
template <int KIND, int NR>
__device__ __forceinline__ void decode(const uint32_t w[NR][2], const uint32_t s[NR], uint32_t o[NR][2][4]) {
  bool two = false;
  if (W4<KIND>::MX) {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < NR; r++) m = max(m, s[r]);
    two = __any_sync(0xffffffffu, m > 128u);
  }
#pragma unroll
  for (int r = 0; r < NR; r++) {
    const uint32_t f = two ? kTwo126 : one_factor<KIND>(s[r]);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      raw_pairs<KIND>(w[r][i], o[r][i]);
#pragma unroll
      for (int j = 0; j < 4; j++) o[r][i][j] = mul_bf16x2(o[r][i][j], f);
    }
  }
  if (W4<KIND>::MX && two) {
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const uint32_t h = w4_scale_bf16x2<KIND>(s[r]);
#pragma unroll
      for (int i = 0; i < 8; i++) o[r][i >> 2][i & 3] = mul_bf16x2(o[r][i >> 2][i & 3], h);
    }
  }
}

__device__ __forceinline__ void mma16816(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Where a lane's column of the mma comes from: one part of one row of a.  A
// part is what is left of the value after the parts before it, each cut to
// bfloat16's bits (an infinity leaves NaN in the later parts, and so in the
// row's results).
template <int DT>
struct Column {
  const uint8_t* row;  // NULL: none
  uint32_t cut0, cut1;
  __device__ __forceinline__ Column(const RowArgs& a, int c) {
    constexpr int P = bf16_parts(DT), ES = DT == DT_F32 ? 4 : 2;
    const int m = c / P, part = c - m * P;
    row = m < a.rows ? reinterpret_cast<const uint8_t*>(a.a) + (int64_t)m * a.lda * ES : nullptr;
    cut0 = part >= 1 ? 0xffff0000u : 0u, cut1 = part >= 2 ? 0xffff0000u : 0u;
  }
  __device__ __forceinline__ uint32_t pair(float a, float b) const {
    a = __fsub_rn(a, __uint_as_float(__float_as_uint(a) & cut0));
    b = __fsub_rn(b, __uint_as_float(__float_as_uint(b) & cut0));
    if (DT == DT_F32) {
      a = __fsub_rn(a, __uint_as_float(__float_as_uint(a) & cut1));
      b = __fsub_rn(b, __uint_as_float(__float_as_uint(b) & cut1));
    }
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  }
  // N elements from column k (zeros from `cols` on), packed in pairs
  template <int N>
  __device__ __forceinline__ void load(int64_t k, int64_t cols, int wide, uint32_t o[N / 2]) const {
#pragma unroll
    for (int i = 0; i < N / 2; i++) o[i] = 0;
    if (!row) return;
    if (wide && k + N <= cols) {
      if (DT == DT_F32) {
        const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k);
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
          const float4 f = __ldg(s + i);
          o[2 * i] = pair(f.x, f.y), o[2 * i + 1] = pair(f.z, f.w);
        }
      } else {
        const uint2* s = reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(row) + k);
        if (N >= 8) {
#pragma unroll
          for (int i = 0; i < N / 8; i++) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(s) + i);
            o[4 * i] = u.x, o[4 * i + 1] = u.y, o[4 * i + 2] = u.z, o[4 * i + 3] = u.w;
          }
        } else {
          const uint2 u = __ldg(s);
          o[0] = u.x, o[1] = u.y;
        }
        if (DT == DT_F16) {
#pragma unroll
          for (int i = 0; i < N / 2; i++) o[i] = pair(f16_bits_to_f32(o[i] & 0xffff), f16_bits_to_f32(o[i] >> 16));
        }
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < N / 2; i++) {
        const int64_t c = k + 2 * i;
        const float a = c < cols ? load_elem(row, DT, c) : 0.0f, b = c + 1 < cols ? load_elem(row, DT, c + 1) : 0.0f;
        const uint32_t v = DT == DT_BF16 ? __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632) : pair(a, b);
#pragma unroll
        for (int j = 0; j < N / 2; j++)  // no register is indexed at run time
          if (j == i) o[j] = v;
      }
    }
  }
};

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

// Adds what `n` floats of WARPS warps (at red + warp * n) and every CTA of the
// cluster hold, always in the same order, and stores `count` results: result
// o is the sum of the `parts` sums at place(o), place(o) + step, ...
template <int WARPS, class Place, class Store>
__device__ __forceinline__ void add_and_store(float* red, int n, int count, int parts, int step, Place&& place,
                                              Store&& store) {
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  __syncthreads();
  if (WARPS > 1) {
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
      float v[WARPS];
#pragma unroll
      for (int w = 0; w < WARPS; w++) v[w] = red[w * n + i];
#pragma unroll
      for (int w = 1; w < WARPS; w++) v[0] = __fadd_rn(v[0], v[w]);
      red[i] = v[0];
    }
    __syncthreads();
  }
  if (ranks > 1) cluster_barrier();
#pragma unroll 1
  for (int o = rank * kRowThreads + threadIdx.x; o < count; o += ranks * kRowThreads) {
    const int at = place(o);
    float sum = 0.0f;
#pragma unroll 1
    for (int p = 0; p < parts; p++) {
      float v = ranks > 1 ? peer_float(red + at + p * step, 0) : red[at + p * step];
#pragma unroll 1
      for (uint32_t r = 1; r < ranks; r++) v = __fadd_rn(v, peer_float(red + at + p * step, r));
      sum = p ? __fadd_rn(sum, v) : v;
    }
    store(o, sum);
  }
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

// x's piece of a step, 256 columns of every row, as bfloat16 parts in shared
// memory: row c of it is column c of the mma, its 256 elements in four runs
// of 64 that lie 144 bytes apart, so that the reads of a quarter warp (two
// columns, four runs) meet no bank twice.
constexpr int kRunPitch = 144, kColPitch = 4 * kRunPitch;
template <int DT, int NT>
struct Piece {
  static constexpr int P = bf16_parts(DT), ROWS = (NT * 8 / P + 3) / 4;  // rows per thread
  static constexpr int BYTES = NT * 8 * kColPitch;
  float v[DT == DT_F32 ? ROWS : 1][4];
  uint2 h[DT == DT_F32 ? 1 : ROWS];
  // four elements of up to ROWS rows: thread t has columns 4 (t % 64) of rows t / 64, t / 64 + 4, ...
  __device__ __forceinline__ void load(const RowArgs& a, int64_t k0) {
    const int64_t k = k0 + (threadIdx.x & 63) * 4;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int m = (threadIdx.x >> 6) + 4 * i;
      const bool on = m < a.rows && k < a.in;
      const int64_t at = (int64_t)m * a.lda + k;
      if (DT == DT_F32) {
        float* d = v[DT == DT_F32 ? i : 0];
        if (on && a.wide && k + 4 <= a.in) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.a) + at));
          d[0] = f.x, d[1] = f.y, d[2] = f.z, d[3] = f.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) d[j] = on && k + j < a.in ? __ldg(reinterpret_cast<const float*>(a.a) + at + j) : 0.0f;
        }
      } else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(a.a) + at;
        uint2 u = make_uint2(0, 0);
        if (on && a.wide && k + 4 <= a.in) {
          u = __ldg(reinterpret_cast<const uint2*>(s));
        } else if (on) {
          u.x = __ldg(s) | (k + 1 < a.in ? (uint32_t)__ldg(s + 1) << 16 : 0u);
          u.y = (k + 2 < a.in ? (uint32_t)__ldg(s + 2) : 0u) | (k + 3 < a.in ? (uint32_t)__ldg(s + 3) << 16 : 0u);
        }
        h[DT == DT_F32 ? 0 : i] = u;
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* buf) const {
    const int e = (threadIdx.x & 63) * 4, at = (e >> 6) * kRunPitch + (e & 63) * 2;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int m = (threadIdx.x >> 6) + 4 * i;
      if ((m + 1) * P > NT * 8) continue;
      uint8_t* d = buf + m * P * kColPitch + at;
      if (DT == DT_BF16) {
        *reinterpret_cast<uint2*>(d) = h[DT == DT_F32 ? 0 : i];
      } else {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
          x[j] = DT == DT_F32 ? v[DT == DT_F32 ? i : 0][j]
                              : f16_bits_to_f32((uint16_t)((j < 2 ? h[DT == DT_F32 ? 0 : i].x : h[DT == DT_F32 ? 0 : i].y) >>
                                                           (16 * (j & 1))));
#pragma unroll
        for (int p = 0; p < P; p++) {
          *reinterpret_cast<uint2*>(d + p * kColPitch) =
              make_uint2(__byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632),
                         __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x7632));
#pragma unroll
          for (int j = 0; j < 4; j++) x[j] = __fsub_rn(x[j], __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u));
        }
      }
    }
  }
};

// y[m, n] for 128 weight rows n per cluster; NT * 8 columns of the mma hold
// rows x parts
template <int NT>
constexpr int kForwardDepth = NT == 4 ? 3 : 4;  // two CTAs per SM
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_forward_kernel(const RowArgs a) {
  using R = Ring<KIND, 256>;
  using X = Piece<DT, NT>;
  constexpr int P = bf16_parts(DT), C = NT * 8, D = kForwardDepth<NT>;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t r0 = (int64_t)(blockIdx.x / cluster_size()) * 128 + warp * kTileR;
  const int64_t steps = (a.in + 255) / 256, stride = cluster_size(), first = cluster_rank();
  uint8_t* const ring = sm + warp * D * R::BYTES;
  uint8_t* const xbuf = sm + kRowWarps * D * R::BYTES;
  float acc[NT][4] = {};
  X x;
  x.load(a, first * 256);
  // columns of the mma that no row fills stay zero
  for (int i = threadIdx.x; i < 2 * X::BYTES / 16; i += kRowThreads) reinterpret_cast<uint4*>(xbuf)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  int slot = 0, turn = 0;
  int64_t ahead = first;
#pragma unroll 1
  for (int64_t s = first - (D - 1) * stride; s < steps; s += stride, ahead += stride, slot = slot + 1 == D ? 0 : slot + 1) {
    __syncwarp();  // all lanes are done with the stage that is filled next
    if (ahead < steps && r0 < a.out) R::fetch(a, ring + slot * R::BYTES, r0, ahead * 256, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (s < 0) continue;
    uint8_t* const xs = xbuf + turn * X::BYTES;
    turn ^= 1;
    x.store(xs);
    x.load(a, (s + stride) * 256);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    __syncthreads();  // the step's x is there, and the last one's has been read
    const uint8_t* const st = ring + (slot + 1 == D ? 0 : slot + 1) * R::BYTES;
    const uint8_t* const p0 = st + R::place(a, r0 + g, s * 256, g);
    const uint8_t* const p1 = st + R::place(a, r0 + g + 8, s * 256, g + 8);
    const int64_t k0 = s * 256 + 64 * t;
#pragma unroll 1
    for (int b = 0; b < 64; b += 16) {
      uint32_t w[2][2], sc[2], o[2][2][4];
      load_run<KIND>(p0, 64 * t + b, w[0], sc[0]);
      load_run<KIND>(p1, 64 * t + b, w[1], sc[1]);
      if (k0 + b >= a.in)  // behind the row's end lie other rows' bytes, or none
        w[0][0] = w[0][1] = w[1][0] = w[1][1] = 0, sc[0] = sc[1] = 56;
      decode<KIND, 2>(w, sc, o);
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const uint4* v = reinterpret_cast<const uint4*>(xs + (n * 8 + g) * kColPitch + t * kRunPitch + b * 2);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const uint4 u = v[i];  // the pairs' order: {1, 5}, {0, 4}, {3, 7}, {2, 6}
          mma16816(acc[n], o[0][i][0], o[1][i][0], o[0][i][1], o[1][i][1], __byte_perm(u.x, u.z, 0x7632),
                   __byte_perm(u.x, u.z, 0x5410));
          mma16816(acc[n], o[0][i][2], o[1][i][2], o[0][i][3], o[1][i][3], __byte_perm(u.y, u.w, 0x7632),
                   __byte_perm(u.y, u.w, 0x5410));
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);  // [weight row][column], an odd pitch
#pragma unroll
  for (int n = 0; n < NT; n++) {
    float* d = red + warp * kTileR * (C + 1) + n * 8 + 2 * t;
    d[g * (C + 1)] = acc[n][0], d[g * (C + 1) + 1] = acc[n][1];
    d[(g + 8) * (C + 1)] = acc[n][2], d[(g + 8) * (C + 1) + 1] = acc[n][3];
  }
  const float scale = __fmul_rn(out_scale(a.o), bias<KIND>());
  const int64_t n0 = r0 - warp * kTileR;
  add_and_store<1>(
      red, 0, 128 * a.rows, P, 1, [&](int o) { return (o & 127) * (C + 1) + (o >> 7) * P; },
      [&](int o, float v) {
        if (n0 + (o & 127) < a.out) finish(a.o, scale, o >> 7, n0 + (o & 127), v);
      });
}

// dx[m, k] for 128 columns k per cluster
constexpr int kDK = 128, kRedPitch = kDK + 8;  // a column's sums: 17 floats per 16 k, so that the eight g's differ in bank
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_dgrad_kernel(const RowArgs a) {
  using R = Ring<KIND, kDK>;
  constexpr int P = bf16_parts(DT), C = NT * 8;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t k0 = (int64_t)(blockIdx.x / cluster_size()) * kDK;
  float acc[8][NT][4] = {};
  uint8_t* const ring = sm + warp * kDepth * R::BYTES;
  const int64_t steps = (a.out + kTileR - 1) / kTileR, stride = (int64_t)kRowWarps * cluster_size();
  int64_t ahead = (int64_t)cluster_rank() * kRowWarps + warp;
  uint32_t y[NT][2];  // of the next step
  int slot = 0;
#pragma unroll
  for (int n = 0; n < NT; n++) Column<DT>(a, n * 8 + g).template load<4>(ahead * kTileR + 4 * t, a.out, a.wide, y[n]);
#pragma unroll 1
  for (int64_t s = ahead - (kDepth - 1) * stride; s < steps; s += stride, ahead += stride, slot = (slot + 1) & (kDepth - 1)) {
    __syncwarp();  // all lanes are done with the stage that is filled next
    if (ahead < steps) R::fetch(a, ring + slot * R::BYTES, ahead * kTileR, k0, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (s < 0) continue;
    uint32_t z[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      z[n][0] = y[n][0], z[n][1] = y[n][1];
      Column<DT>(a, n * 8 + g).template load<4>((s + stride) * kTileR + 4 * t, a.out, a.wide, y[n]);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    __syncwarp();
    const uint8_t* const st = ring + ((slot + 1) & (kDepth - 1)) * R::BYTES;
    const int64_t n0 = s * kTileR + 4 * t;
    uint32_t w[4][2], sc[4], o[4][2][4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      load_run<KIND>(st + R::place(a, n0 + r, k0, 4 * t + r), 16 * g, w[r], sc[r]);
      if (n0 + r >= a.out) w[r][0] = w[r][1] = 0, sc[r] = 56;  // behind the last row: whatever the stage held
    }
    decode<KIND, 4>(w, sc, o);
#pragma unroll
    for (int q = 0; q < 8; q++) {
      const int i = q >> 2, j = q & 3;
      const uint32_t a0 = __byte_perm(o[0][i][j], o[1][i][j], 0x5410), a1 = __byte_perm(o[0][i][j], o[1][i][j], 0x7632);
      const uint32_t a2 = __byte_perm(o[2][i][j], o[3][i][j], 0x5410), a3 = __byte_perm(o[2][i][j], o[3][i][j], 0x7632);
#pragma unroll
      for (int n = 0; n < NT; n++) mma16816(acc[q][n], a0, a1, a2, a3, z[n][0], z[n][1]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(sm);  // [warp][column][17 floats per 16 k]
#pragma unroll
  for (int q = 0; q < 8; q++) {
    // the pair's two weights: {1, 5}, {0, 4}, {3, 7}, {2, 6} of word q / 4
    constexpr int first[4] = {1, 0, 3, 2};
    const int e = (q >> 2) * 8 + first[q & 3];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float* d = red + (warp * C + n * 8 + 2 * t) * kRedPitch + 17 * g + e;
      d[0] = acc[q][n][0], d[kRedPitch] = acc[q][n][1];
      d[4] = acc[q][n][2], d[kRedPitch + 4] = acc[q][n][3];
    }
  }
  const float scale = __fmul_rn(out_scale(a.o), bias<KIND>());
  add_and_store<kRowWarps>(
      red, C * kRedPitch, kDK * a.rows, P, kRedPitch,
      [&](int o) { return (o >> 7) * P * kRedPitch + 17 * ((o & 127) >> 4) + (o & 15); },
      [&](int o, float v) {
        if (k0 + (o & 127) < a.in) finish(a.o, scale, o >> 7, k0 + (o & 127), v);
      });
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

template <void (*kernel)(const RowArgs)>
cudaError_t launch_rows(const RowArgs& a, int64_t tiles, int64_t steps, int smem, int sms, cudaStream_t st) {
  // up to two CTAs per SM while each still has a step to do
  int cluster = 1;
  while (cluster < 8 && tiles * cluster * 2 <= 2 * sms && cluster < steps) cluster *= 2;
  static bool set[64] = {false};  // of this kernel, per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
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
    return launch_rows<rows_forward_kernel<KIND, DT, NT>>(
        a, (a.out + 127) / 128, (a.in + 255) / 256,
        kRowWarps * kForwardDepth<NT> * Ring<KIND, 256>::BYTES + 2 * Piece<DT, NT>::BYTES, sms, st);
  if constexpr (NT <= 2)
    return launch_rows<rows_dgrad_kernel<KIND, DT, NT>>(
        a, (a.in + kDK - 1) / kDK, (a.out + kRowWarps * kTileR - 1) / (kRowWarps * kTileR),
        std::max(kRowWarps * kDepth * Ring<KIND, kDK>::BYTES, kRowWarps * NT * 8 * kRedPitch * 4), sms, st);
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
