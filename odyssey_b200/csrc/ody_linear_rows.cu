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
//   forward: rows g and g + 8 of the 16 (g = lane / 4), columns 16 t to 16 t
//            + 15 of every 64 (t = lane % 4); the reduction is over columns
//   dgrad:   rows 4 t to 4 t + 3, columns 16 g to 16 g + 15; the reduction is
//            over rows, so neighbouring rows are paired by byte permutes
// Eight warps share the reduction, and a cluster of up to eight CTAs where
// the outputs alone do not fill the GPU; their sums are added in a fixed
// order through (distributed) shared memory.  One launch, no workspace.
// (Sixteen warps on 256 weight rows that share x's piece, with clusters for
// the columns, took 27 us for one row x 4096^2: clusters of eight CTAs that
// need an SM each leave most SMs idle.)
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

constexpr int kRowThreads = 256, kRowWarps = 8, kTileR = 16, kDepth = 3;  // kDepth: dgrad's stages

struct RowArgs {
  LinearOut o;
  const void* a;  // x or dy
  int64_t lda;
  const uint8_t* q;
  int64_t out, in;  // weight rows and columns
  int rows;         // of a
  int wide;         // a's rows are 16-byte aligned
  int keep;         // dgrad: a warp has more than 32 steps
};

// A warp's ring of weight tiles, 16 rows x K columns each.  A row's piece is
// at most K * 9 / 16 bytes at any byte offset, so it is copied as the aligned
// 16-byte words around it.  For 256 columns the pitch of eleven words keeps a
// warp's reads, eight rows by four offsets of nine words, on 32 banks.
template <int KIND, int K>
struct Ring {
  using W = W4<KIND>;
  static constexpr int WORDS = (K * 9 / 16 + 30) / 16, PITCH = (WORDS | 1) * 16, BYTES = kTileR * PITCH;
  static constexpr int AT_ONCE = 32 / WORDS;  // rows that one copy of every lane takes
  static_assert(K % 128 == 0, "whole blocks");

  // Columns k0.. of rows r0.. into a stage; neighbouring lanes copy
  // neighbouring words of a row (two lanes to a row, each with every other
  // word, halved the rate).  What lies behind a row's end comes as zeros, so
  // nothing is read past the weight; a word that begins before the weight is
  // copied byte by byte.
  static __device__ __forceinline__ void fetch(const RowArgs& a, uint8_t* st, int64_t r0, int k0, int lane) {
    const uint32_t row_bytes = (uint32_t)(a.in / W::BE * W::SB);
    const int r = lane / WORDS, w = lane - r * WORDS;
    if (r >= AT_ONCE) return;
    const uint32_t left = row_bytes - k0 / W::BE * W::SB;  // of a row, from k0 on
    uintptr_t src = reinterpret_cast<uintptr_t>(a.q + (r0 + r) * row_bytes + k0 / W::BE * W::SB) + w * 16;
    uint32_t d = srow(st) + r * PITCH + w * 16;
    if (r0 + kTileR <= a.out && left >= WORDS * 16 && (r0 > 0 || k0 > 0)) {
#pragma unroll
      for (int i = 0; i < kTileR; i += AT_ONCE, src += AT_ONCE * row_bytes)
        if (i + AT_ONCE <= kTileR || i + r < kTileR)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + i * PITCH), "l"(src & ~(uintptr_t)15) : "memory");
    } else {
#pragma unroll 1
      for (int i = r; i < kTileR && r0 + i < a.out; i += AT_ONCE, src += AT_ONCE * row_bytes, d += AT_ONCE * PITCH) {
        const uintptr_t p = src & ~(uintptr_t)15;
        const int64_t n = (int64_t)(reinterpret_cast<uintptr_t>(a.q) + (r0 + i + 1) * row_bytes) - (int64_t)p;  // to the row's end
        if (p >= reinterpret_cast<uintptr_t>(a.q)) {
          const uint32_t size = n >= 16 ? 16 : (n > 0 ? (uint32_t)n : 0);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(size ? p : reinterpret_cast<uintptr_t>(a.q)),
                       "r"(size)
                       : "memory");
        } else {
          uint8_t* const e = st + i * PITCH + w * 16;
#pragma unroll 1
          for (int b = 0; b < 16; b++)
            e[b] = b < n && p + b >= reinterpret_cast<uintptr_t>(a.q) ? *reinterpret_cast<const uint8_t*>(p + b) : 0;
        }
      }
    }
  }
};

// Tables in shared memory: a code byte as its two weights in bfloat16, one
// copy per lane so that no two lanes meet in a bank (entry b of lane l at 128
// b + 4 l), and a block's scale byte as a bfloat16 pair.  Per pair of weights
// that leaves a byte extraction, an address, one load and the multiplication
// by the scale, spread over four pipes; with integer operations alone (5 per
// pair on the half-rate pipe) 8 rows x 8192^2 took 32 us.
constexpr int kTableBytes = 256 * 128 + 256 * 4;
template <int KIND>
__device__ __forceinline__ void make_tables(uint8_t* table) {
  static_assert(kRowThreads == 256, "a thread per entry");
  const int e = threadIdx.x;
  const uint32_t pair = __byte_perm(__float_as_uint(W4<KIND>::value(e >> 4, 1.0f)),
                                    __float_as_uint(W4<KIND>::value(e & 15, 1.0f)), 0x7632);
  uint4* d = reinterpret_cast<uint4*>(table + e * 128);
#pragma unroll
  for (int i = 0; i < 8; i++) d[(i + e) & 7] = make_uint4(pair, pair, pair, pair);  // turned, so that lanes differ in bank
  reinterpret_cast<uint32_t*>(table + 256 * 128)[e] = w4_scale_bf16x2<KIND>(e);
}

// word at a byte offset of shared memory (a multiple of four)
__device__ __forceinline__ uint32_t word(const uint8_t* sm, uint32_t at) {
  return *reinterpret_cast<const uint32_t*>(sm + at);
}
__device__ __forceinline__ uint32_t shift_down(uint32_t lo, uint32_t hi, uint32_t bits) {  // bits taken mod 32
  return __funnelshift_r(lo, hi, bits);
}

// Where sixteen weights of a row lie in shared memory: the aligned word their
// codes begin in and the shift that brings them down; for 32-element blocks
// their block's scale byte.
struct At16 {
  uint32_t word, shift, scale;
};
// block: the block's first byte, half: the byte of its codes to begin with
// (0, or 8 in the second half of 32)
__device__ __forceinline__ At16 at16(uint32_t block, uint32_t half) {
  return {(block + half) & ~3u, (block + half) * 8, block + 16};
}
// their two code words and scale (as a bfloat16 pair), `ahead` bytes further on
template <int KIND>
__device__ __forceinline__ void load16(const uint8_t* sm, const At16& at, uint32_t ahead, uint32_t w[2], uint32_t& f) {
  const uint32_t v0 = word(sm, at.word + ahead), v1 = word(sm, at.word + ahead + 4), v2 = word(sm, at.word + ahead + 8);
  const uint32_t sb = W4<KIND>::MX ? sm[at.scale + ahead] : shift_down(v2, 0, at.shift) & 0xffu;
  w[0] = shift_down(v0, v1, at.shift), w[1] = shift_down(v1, v2, at.shift);
  f = word(sm, 256 * 128 + sb * 4);
}
// the sixteen weights of two code words, o[i] = weights 2 i and 2 i + 1;
// lane4: four times this lane's number
__device__ __forceinline__ void decode16(const uint8_t* sm, uint32_t lane4, uint32_t w0, uint32_t w1, uint32_t f,
                                         uint32_t o[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t b = __byte_perm(i < 4 ? w0 : w1, 0, 0x4440 + (i & 3));
    o[i] = mul_bf16x2(word(sm, b * 128 + lane4), f);
  }
}

// Where a lane's column of the mma comes from: one part of one row of a (of
// row 0 where there is none; nobody reads such a column's results).  A part
// is what is left of the value after the parts before it, each cut to
// bfloat16's bits (an infinity leaves NaN in the later parts, and so in the
// row's results).
template <int DT>
struct Column {
  const uint8_t* row;
  uint32_t cut0, cut1;
  __device__ __forceinline__ void set(const RowArgs& a, int c) {
    constexpr int P = bf16_parts(DT), ES = DT == DT_F32 ? 4 : 2;
    const int m = c / P, part = c - m * P;
    row = reinterpret_cast<const uint8_t*>(a.a) + (m < a.rows ? (int64_t)m * a.lda * ES : 0);
    cut0 = part >= 1 ? 0xffff0000u : 0u, cut1 = part >= 2 ? 0xffff0000u : 0u;
  }
  __device__ __forceinline__ uint32_t pair(float a, float b) const {
    if (DT != DT_BF16) {
      a = __fsub_rn(a, __uint_as_float(__float_as_uint(a) & cut0));
      b = __fsub_rn(b, __uint_as_float(__float_as_uint(b) & cut0));
    }
    if (DT == DT_F32) {
      a = __fsub_rn(a, __uint_as_float(__float_as_uint(a) & cut1));
      b = __fsub_rn(b, __uint_as_float(__float_as_uint(b) & cut1));
    }
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  }
  // sixteen elements from index k, packed in pairs; all: they are there and
  // 16-byte aligned, else zeros from `n` on
  __device__ __forceinline__ void load16(int k, int n, bool all, uint32_t o[8]) const {
    if (all) {
      if (DT == DT_F32) {
        const float4* s = reinterpret_cast<const float4*>(row + (uint32_t)k * 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4 f = __ldg(s + i);
          o[2 * i] = pair(f.x, f.y), o[2 * i + 1] = pair(f.z, f.w);
        }
      } else {
        const uint4* s = reinterpret_cast<const uint4*>(row + (uint32_t)k * 2);
        const uint4 u = __ldg(s), v = __ldg(s + 1);
        o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w, o[4] = v.x, o[5] = v.y, o[6] = v.z, o[7] = v.w;
        if (DT == DT_F16) {
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] = pair(f16_bits_to_f32(o[i] & 0xffff), f16_bits_to_f32(o[i] >> 16));
        }
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < 8; i++) {
        const float f0 = k + 2 * i < n ? load_elem(row, DT, k + 2 * i) : 0.0f;
        const float f1 = k + 2 * i + 1 < n ? load_elem(row, DT, k + 2 * i + 1) : 0.0f;
        const uint32_t v = pair(f0, f1);
#pragma unroll
        for (int j = 0; j < 8; j++)  // no register is indexed at run time
          if (j == i) o[j] = v;
      }
    }
  }
  // four elements from index k (zeros from `n` on), packed in pairs
  __device__ __forceinline__ void load(int64_t k, int64_t n, int wide, uint32_t o[2]) const {
    o[0] = o[1] = 0;
    if (k >= n) return;
    if (wide && k + 4 <= n) {
      if (DT == DT_F32) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k));
        o[0] = pair(f.x, f.y), o[1] = pair(f.z, f.w);
      } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(row) + k));
        o[0] = u.x, o[1] = u.y;
        if (DT == DT_F16) {
          o[0] = pair(f16_bits_to_f32(u.x & 0xffff), f16_bits_to_f32(u.x >> 16));
          o[1] = pair(f16_bits_to_f32(u.y & 0xffff), f16_bits_to_f32(u.y >> 16));
        }
      }
    } else {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = k + i < n ? load_elem(row, DT, k + i) : 0.0f;
      o[0] = pair(f[0], f[1]), o[1] = pair(f[2], f[3]);
    }
  }
};

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
      float v[8];
      if (ranks == 1) {
        v[0] = red[at + p * step];
      } else {
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) v[r] = r < ranks ? peer_float(red + at + p * step, r) : 0.0f;
#pragma unroll
        for (uint32_t r = 1; r < 8; r++) v[0] = __fadd_rn(v[0], v[r]);
      }
      sum = p ? __fadd_rn(sum, v[0]) : v[0];
    }
    store(o, sum);
  }
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

// y[m, n]: a CTA (or cluster) takes 16 weight rows n at a time, every
// gridDim.x / cluster-th such tile; NT * 8 columns of the mma hold rows x
// parts.  The weight's bytes of the next tile are under way while a tile's
// sums are added.
template <int NT>
constexpr int kForwardDepth = NT == 4 ? 2 : 3;  // two CTAs per SM
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_forward_kernel(const RowArgs a) {
  using W = W4<KIND>;
  using R = Ring<KIND, 256>;
  constexpr int P = bf16_parts(DT), C = NT * 8, kDepth = kForwardDepth<NT>;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const ring = sm + kTableBytes + warp * kDepth * R::BYTES;
  float* const red = reinterpret_cast<float*>(sm + kTableBytes + kRowWarps * kDepth * R::BYTES);
  const int in = (int)a.in, steps = (in + 255) / 256, stride = kRowWarps * (int)cluster_size();
  const int me = (int)cluster_rank() * kRowWarps + warp;
  const int mine = me < steps ? (steps - me + stride - 1) / stride : 0;  // this warp's steps of a tile
  const int64_t tiles = (a.out + kTileR - 1) / kTileR, tile_stride = gridDim.x / cluster_size();
  int64_t tile = blockIdx.x / cluster_size();
  make_tables<KIND>(sm);
  const uint32_t lane4 = lane * 4, at0 = kTableBytes + warp * kDepth * R::BYTES + g * R::PITCH + 16 * t / W::BE * W::SB;
  const uint32_t half = 16 * t % W::BE / 2;  // this lane's 16 of every 64 columns: a block, or half a block of 32
  const uint32_t q0 = (uint32_t)reinterpret_cast<uintptr_t>(a.q), row_bytes = (uint32_t)(a.in / W::BE * W::SB);
  const float scale = out_scale(a.o);
  Column<DT> cols[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) cols[n].set(a, n * 8 + g);
  // what is fetched next: step fs (of `mine`) of tile ft
  int64_t ft = tile;
  int fs = 0, slot = 0;
  const auto fetch = [&](int to) {
    if (fs < mine && ft < tiles) R::fetch(a, ring + to * R::BYTES, ft * kTileR, (me + fs * stride) * 256, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++fs >= mine) fs = 0, ft += tile_stride;
  };
#pragma unroll 1
  for (int i = 0; i < kDepth - 1; i++) fetch(i);
  // the next run's 16 elements of the columns' rows (zeros behind the rows' end)
  uint32_t x[2][NT][8];
  const auto load_x = [&](int k, uint32_t (*o)[8]) {
    const bool all = a.wide && k + 16 <= in;
#pragma unroll
    for (int n = 0; n < NT; n++) cols[n].load16(k, in, all, o[n]);
  };
  load_x(me * 256 + 16 * t, x[0]);
  __syncthreads();
#pragma unroll 1
  for (; tile < tiles; tile += tile_stride) {
    const int64_t r0 = tile * kTileR;
    const uint32_t sk0 = q0 + (uint32_t)(r0 + g) * row_bytes, sk1 = sk0 + 8 * row_bytes;
    float acc[NT][4] = {}, part[NT][4] = {};  // part: of two steps, 32 mma (a tensor core cuts low bits off)
#pragma unroll 1
    for (int i = 0; i < mine; i++) {
      const int s = me + i * stride, k0 = s * 256 + 16 * t;
      const int next = i + 1 < mine ? k0 + stride * 256 : me * 256 + 16 * t;  // where the step after this one begins
      __syncwarp();  // all lanes are done with the stage that is filled next
      fetch(slot == 0 ? kDepth - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();
      const uint32_t adv = (uint32_t)s * (256 / W::BE * W::SB), off = at0 + slot * R::BYTES;
      slot = slot + 1 == kDepth ? 0 : slot + 1;
      // 64 columns are 34 or 36 bytes, 128 a multiple of four: two places a row
      constexpr uint32_t RUN = 64 / W::BE * W::SB;
      const uint32_t p0 = off + ((sk0 + adv) & 15u), p1 = off + 8 * R::PITCH + ((sk1 + adv) & 15u);
      const At16 e0[2] = {at16(p0, half), at16(p0 + RUN, half)}, e1[2] = {at16(p1, half), at16(p1 + RUN, half)};
#pragma unroll 1
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          load_x(b + h < 2 ? k0 + 128 * b + 64 * h + 64 : next, x[1 - h]);
          uint32_t w0[2], w1[2], f0, f1, o0[8], o1[8];
          load16<KIND>(sm, e0[h], 2 * RUN * b, w0, f0);
          load16<KIND>(sm, e1[h], 2 * RUN * b, w1, f1);
          decode16(sm, lane4, w0[0], w0[1], f0, o0);
          decode16(sm, lane4, w1[0], w1[1], f1, o1);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              mma16816(part[n], o0[j], o1[j], o0[j + 1], o1[j + 1], x[h][n][j], x[h][n][j + 1]);
        }
      if ((i & 1) || i + 1 == mine) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[n][j] = __fadd_rn(acc[n][j], part[n][j]), part[n][j] = 0.0f;
      }
    }
    // red: [warp][weight row][column], an odd pitch
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float* d = red + warp * kTileR * (C + 1) + n * 8 + 2 * t;
      d[g * (C + 1)] = acc[n][0], d[g * (C + 1) + 1] = acc[n][1];
      d[(g + 8) * (C + 1)] = acc[n][2], d[(g + 8) * (C + 1) + 1] = acc[n][3];
    }
    add_and_store<kRowWarps>(
        red, kTileR * (C + 1), kTileR * a.rows, P, 1, [&](int o) { return (o & 15) * (C + 1) + (o >> 4) * P; },
        [&](int o, float v) {
          if (r0 + (o & 15) < a.out) finish(a.o, scale, o >> 4, r0 + (o & 15), v);
        });
    __syncthreads();  // red is free again
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// dx[m, k] for 128 columns k per cluster
constexpr int kDK = 128, kRedPitch = kDK + 8;  // a column's sums: 17 floats per 16 k, so that the eight g's differ in bank
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_dgrad_kernel(const RowArgs a) {
  using W = W4<KIND>;
  using R = Ring<KIND, kDK>;
  constexpr int P = bf16_parts(DT), C = NT * 8;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t k0 = (int64_t)(blockIdx.x / cluster_size()) * kDK;
  const int64_t steps = (a.out + kTileR - 1) / kTileR, stride = (int64_t)kRowWarps * cluster_size();
  uint8_t* const ring = sm + kTableBytes + warp * kDepth * R::BYTES;
  // A warp's sums, [column][17 floats per 16 k].  Where it has more than 32
  // steps they have a place of their own and take the accumulators in every
  // 32 mma (a tensor core cuts low bits off); else they lie where the ring was.
  float* const sums = reinterpret_cast<float*>(sm + (a.keep ? kTableBytes + kRowWarps * kDepth * R::BYTES : 0));
  int64_t ahead = (int64_t)cluster_rank() * kRowWarps + warp;
  uint32_t y[NT][2];  // of the next step
  Column<DT> cols[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    cols[n].set(a, n * 8 + g);
    cols[n].load(ahead * kTileR + 4 * t, a.out, a.wide, y[n]);
  }
  make_tables<KIND>(sm);
  __syncthreads();
  const uint32_t q0 = (uint32_t)reinterpret_cast<uintptr_t>(a.q), row_bytes = (uint32_t)(a.in / W::BE * W::SB);
  const uint32_t sk = q0 + (uint32_t)(k0 / W::BE) * W::SB;
  // this lane's 16 columns: a block, or half a block of 32
  const uint32_t at0 = kTableBytes + warp * kDepth * R::BYTES + 16 * g / W::BE * W::SB, half = 16 * g % W::BE / 2;
  int slot = 0;
  int64_t s = ahead - (kDepth - 1) * stride;
  bool first = true;
#pragma unroll 1
  do {
    float acc[8][NT][4] = {};
    const int64_t end = a.keep ? min(steps, s + 32 * stride) : steps;
#pragma unroll 1
    for (; s < end; s += stride, ahead += stride, slot = slot + 1 == kDepth ? 0 : slot + 1) {
      __syncwarp();  // all lanes are done with the stage that is filled next
      if (ahead < steps) R::fetch(a, ring + slot * R::BYTES, ahead * kTileR, (int)k0, lane);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (s < 0) continue;
      uint32_t z[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        z[n][0] = y[n][0], z[n][1] = y[n][1];
        cols[n].load((s + stride) * kTileR + 4 * t, a.out, a.wide, y[n]);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      __syncwarp();
      const uint32_t st = at0 + (slot + 1 == kDepth ? 0 : slot + 1) * R::BYTES;
      const int64_t n0 = s * kTileR + 4 * t;
      uint32_t o[4][8];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t block = st + (4 * t + r) * R::PITCH + ((sk + (uint32_t)(n0 + r) * row_bytes) & 15u);
        uint32_t w[2], f;
        load16<KIND>(sm, at16(block, half), 0, w, f);
        if (n0 + r >= a.out) w[0] = w[1] = f = 0;  // behind the last row: whatever the stage held
        decode16(sm, lane * 4, w[0], w[1], f, o[r]);
      }
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const uint32_t a0 = __byte_perm(o[0][q], o[1][q], 0x5410), a1 = __byte_perm(o[0][q], o[1][q], 0x7632);
        const uint32_t a2 = __byte_perm(o[2][q], o[3][q], 0x5410), a3 = __byte_perm(o[2][q], o[3][q], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; n++) mma16816(acc[q][n], a0, a1, a2, a3, z[n][0], z[n][1]);
      }
    }
    if (s >= steps) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < 8; q++)
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float* d = sums + (warp * C + n * 8 + 2 * t) * kRedPitch + 17 * g + 2 * q;
        float* const at[4] = {d, d + kRedPitch, d + 1, d + kRedPitch + 1};
#pragma unroll
        for (int i = 0; i < 4; i++) *at[i] = first ? acc[q][n][i] : __fadd_rn(*at[i], acc[q][n][i]);
      }
    first = false;
  } while (s < steps);
  const float scale = out_scale(a.o);
  add_and_store<kRowWarps>(
      sums, C * kRedPitch, kDK * a.rows, P, kRedPitch,
      [&](int o) { return (o >> 7) * P * kRedPitch + 17 * ((o & 127) >> 4) + (o & 15); },
      [&](int o, float v) {
        if (k0 + (o & 127) < a.in) finish(a.o, scale, o >> 7, k0 + (o & 127), v);
      });
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

// CTAs that share a tile: two per SM are launched, and fewer tiles than that
// are shared while every CTA still has a step for its warps
int cluster_for(int64_t tiles, int64_t steps, int sms) {
  int cluster = 1;
  while (cluster < 8 && tiles * cluster * 2 <= 2 * sms && cluster < steps) cluster *= 2;
  return cluster;
}

template <void (*kernel)(const RowArgs)>
cudaError_t launch_rows(const RowArgs& a, int64_t grid, int cluster, int smem, cudaStream_t st) {
  static int most[64] = {0};  // of this kernel, per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || most[dev] < smem) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) most[dev] = smem;
  }
  if (cluster == 1) {
    kernel<<<(unsigned)grid, kRowThreads, smem, st>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(grid * cluster));
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
cudaError_t launch_one(const LinearArgs& l, RowArgs a, int sms, cudaStream_t st) {
  const int64_t rows = (a.out + kTileR - 1) / kTileR;
  if (l.op == LIN_FORWARD) {
    const int cluster = cluster_for(rows, (a.in + 256 * kRowWarps - 1) / (256 * kRowWarps), sms);
    return launch_rows<rows_forward_kernel<KIND, DT, NT>>(
        a, std::min<int64_t>(rows, 2 * sms), cluster,
        kTableBytes + kRowWarps * kForwardDepth<NT> * Ring<KIND, 256>::BYTES + kRowWarps * kTileR * (NT * 8 + 1) * 4, st);
  }
  if constexpr (NT <= 2) {
    constexpr int ring = kTableBytes + kRowWarps * kDepth * Ring<KIND, kDK>::BYTES, sums = kRowWarps * NT * 8 * kRedPitch * 4;
    const int64_t tiles = (a.in + kDK - 1) / kDK;
    const int cluster = cluster_for(tiles, (rows + kRowWarps - 1) / kRowWarps, sms);
    a.keep = rows > 32 * (int64_t)kRowWarps * cluster;
    return launch_rows<rows_dgrad_kernel<KIND, DT, NT>>(a, tiles, cluster, a.keep ? ring + sums : std::max(ring, sums), st);
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
  a.keep = 0;
  a.wide = (reinterpret_cast<uintptr_t>(l.a) & 15u) == 0 && (l.rows == 1 || (l.lda * (l.a_dtype == DT_F32 ? 4 : 2)) % 16 == 0);
  if (l.kind == Q_MXFP4) return launch_dt<Q_MXFP4>(l, a, sms, st);
  if (l.kind == Q_MXFP4_OCP) return launch_dt<Q_MXFP4_OCP>(l, a, sms, st);
  return launch_dt<Q_NVFP4>(l, a, sms, st);
}

}  // namespace ody
