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
  int cluster;      // forward: log2 of the CTAs of a cluster,
  int per, extra;   // rows / 8 of a cluster's run, and how many runs have one more
};

// A warp's ring of weight tiles, ROWS rows x K columns each.  A row's piece is
// at most K * 9 / 16 bytes at any byte offset, so it is copied as the aligned
// 16-byte words around it.  An odd pitch in words spreads a warp's reads,
// eight rows by four offsets, over the banks.
template <int KIND, int K, int ROWS>
struct Ring {
  using W = W4<KIND>;
  static constexpr int WORDS = (K * 9 / 16 + 30) / 16, PITCH = (WORDS | 1) * 16, BYTES = ROWS * PITCH;
  static constexpr int AT_ONCE = 32 / WORDS;  // rows that one copy of every lane takes
  static_assert(K % 128 == 0, "whole blocks");

  // where this lane's row and word of rows r0.. begin
  static __device__ __forceinline__ uintptr_t place(const RowArgs& a, int64_t r0, int lane) {
    return reinterpret_cast<uintptr_t>(a.q) + (r0 + lane / WORDS) * (a.in / W::BE * W::SB) + lane % WORDS * 16;
  }
  // Columns k0.. (`before` bytes into their rows) of n rows r0.. into a stage,
  // from place(r0); neighbouring lanes copy neighbouring words of a row (two
  // lanes to a row, each with every other word, halved the rate).  What lies
  // behind a row's end comes as zeros where its columns are used, so nothing
  // is read past the weight; a word that begins before the weight is copied
  // byte by byte.
  static __device__ __forceinline__ void fetch(const RowArgs& a, uint8_t* st, uintptr_t from, int r0, int n, int k0,
                                               uint32_t before, int lane) {
    const uint32_t row_bytes = (uint32_t)(a.in / W::BE * W::SB);
    const uint64_t more = (uint64_t)AT_ONCE * row_bytes;
    const int r = lane / WORDS;
    if (r >= AT_ONCE) return;
    const uintptr_t q = reinterpret_cast<uintptr_t>(a.q);
    from += before;
    uint32_t d = srow(st) + r * PITCH + lane % WORDS * 16;
    if (k0 <= (int)a.in - K && (r0 + n < (int)a.out || before + WORDS * 16 <= row_bytes) && ((q & 15) == 0 || (r0 | k0) != 0)) {
      const int have = n - r;
#pragma unroll
      for (int i = 0; i < ROWS; i += AT_ONCE, from += more)
        if (i < have)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + i * PITCH), "l"(from & ~(uintptr_t)15) : "memory");
    } else {
#pragma unroll 1
      for (int i = r; i < n; i += AT_ONCE, from += more, d += AT_ONCE * PITCH) {
        const uintptr_t p = from & ~(uintptr_t)15;
        const int64_t to_end = (int64_t)(q + (uint64_t)(r0 + i + 1) * row_bytes) - (int64_t)p;  // of the row
        if (p >= q) {
          const uint32_t size = to_end >= 16 ? 16 : (to_end > 0 ? (uint32_t)to_end : 0);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(size ? p : q & ~(uintptr_t)15), "r"(size) : "memory");
        } else {
          uint8_t* const e = st + i * PITCH + lane % WORDS * 16;
#pragma unroll 1
          for (int b = 0; b < 16; b++) e[b] = b < to_end && p + b >= q ? *reinterpret_cast<const uint8_t*>(p + b) : 0;
        }
      }
    }
  }
};

// Weights come from tables in shared memory or by byte permutes.  Tables: a
// code byte as its two weights in bfloat16 and a block's scale byte as a
// bfloat16 pair, one copy per lane so that no two lanes meet in a bank: entry
// b of lane l at 256 b + 4 l, scales 128 further on.  With that stride one
// byte permute puts a byte and the lane together as an address, so a pair of
// weights takes a permute, a load and the multiplication by the scale.
// Without them only the scales have a table, of one copy, and a pair takes
// four permutes and logical operations and the multiplication.  With tables
// the bound is shared memory's one access a cycle (8 rows x 8192^2: 15.8
// accesses a warp for 16 weights of a lane, half of them look-ups), without
// them the integer pipes: 20.5 us against 21.7, one row x 4096^2 6.6 against
// 7.4, the backward product of 4 float32 rows x 4096^2 13.4 against 14.8.
// From 16 columns of the mma on there is no room for two CTAs' tables (one
// CTA of 16 rows x 8192^2 with them took 32.5 us, two without 26.3).
template <bool TABLES>
constexpr int kTableBytes = TABLES ? 256 * 256 : 256 * 4;
template <int KIND, bool TABLES>
__device__ __forceinline__ void make_tables(uint8_t* table) {
  static_assert(kRowThreads == 256, "a thread per entry");
  const int e = threadIdx.x;
  const uint32_t scale = w4_scale_bf16x2<KIND>(e);
  if (!TABLES) {
    reinterpret_cast<uint32_t*>(table)[e] = scale;
    return;
  }
  uint32_t raw[4];
  w4_raw8<KIND>(e, raw);
  const uint32_t pair = mul_bf16x2(raw[0], kTwo126);
  uint4* d = reinterpret_cast<uint4*>(table + e * 256);
#pragma unroll
  for (int i = 0; i < (KIND == Q_MXFP4 ? 8 : 16); i++) {  // E8M0's scales without zero and NaN take no table
    const uint32_t v = i < 8 ? pair : scale;
    d[(i & 8) | ((i + e) & 7)] = make_uint4(v, v, v, v);  // turned, so that lanes differ in bank
  }
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
// byte i of w as the place of this lane's table entry; lane4: four times the lane's number
__device__ __forceinline__ uint32_t entry(uint32_t w, int i, uint32_t lane4) { return __byte_perm(w, lane4, 0x5504 + 16 * i); }
// their two code words and scale (as a bfloat16 pair), `ahead` bytes further on
template <int KIND, bool TABLES>
__device__ __forceinline__ void load16(const uint8_t* sm, const At16& at, uint32_t ahead, uint32_t lane4, uint32_t w[2],
                                       uint32_t& f) {
  const uint32_t v0 = word(sm, at.word + ahead), v1 = word(sm, at.word + ahead + 4), v2 = word(sm, at.word + ahead + 8);
  const uint32_t sb = W4<KIND>::MX ? sm[at.scale + ahead] : shift_down(v2, 0, at.shift);  // in the lowest byte
  w[0] = shift_down(v0, v1, at.shift), w[1] = shift_down(v1, v2, at.shift);
  if (KIND == Q_MXFP4)
    f = sb * 0x00800080u;  // the byte is a bfloat16's exponent
  else
    f = word(sm, TABLES ? entry(sb, 0, lane4) + 128 : (sb & 0xffu) * 4);
}
// the eight weights of a code word, o[i] = weights 2 i and 2 i + 1: from the table
__device__ __forceinline__ void look_up(const uint8_t* sm, uint32_t lane4, uint32_t w, uint32_t f, uint32_t o[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = mul_bf16x2(word(sm, entry(w, i, lane4)), f);
}
// and by byte permutes alone: a permute looks four magnitudes' high bytes up
// in eight, one their low bytes, and one spreads their signs (a selector's
// highest bit repeats the sign of the byte, 0x80, so 0x80 or 0xff)
template <int KIND>
__device__ __forceinline__ void permute(uint32_t w, uint32_t f, uint32_t o[4]) {
  constexpr uint32_t half = KIND == Q_MXFP4_OCP ? 0x3f00u : 0u;  // code 1
  const uint32_t mag = w & 0x77777777u;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t hi = __byte_perm(0x3f3f0000u | half, 0x40404040u, mag >> 16 * i);
    const uint32_t lo = __byte_perm(0xc0800000u, 0xc0804000u, mag >> 16 * i);
    uint32_t sg;
    asm("prmt.b32 %0, %1, %1, %2;" : "=r"(sg) : "r"(0x80808080u), "r"(w >> 16 * i));
    const uint32_t h = hi | (sg << 1 & 0x80808080u);
    o[2 * i] = mul_bf16x2(__byte_perm(lo, h, 0x4051), f);
    o[2 * i + 1] = mul_bf16x2(__byte_perm(lo, h, 0x6273), f);
  }
}
// the sixteen of two
template <int KIND, bool TABLES>
__device__ __forceinline__ void decode16(const uint8_t* sm, uint32_t lane4, uint32_t w0, uint32_t w1, uint32_t f,
                                         uint32_t o[8]) {
  if (TABLES) {
    look_up(sm, lane4, w0, f, o);
    look_up(sm, lane4, w1, f, o + 4);
  } else {
    permute<KIND>(w0, f, o);
    permute<KIND>(w1, f, o + 4);
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
        const float4* s = reinterpret_cast<const float4*>(row + (uint64_t)(uint32_t)k * 4);
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

// Adds what `n` floats of the eight warps (at red + warp * n) and every CTA of the
// cluster hold, always in the same order, and stores `count` results: result
// o is the sum of the `parts` sums at place(o), place(o) + step, ...
template <class Place, class Store>
__device__ __forceinline__ void add_and_store(float* red, int n, int count, int parts, int step, Place&& place,
                                              Store&& store) {
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kRowThreads) {
    float v[kRowWarps];
#pragma unroll
    for (int w = 0; w < kRowWarps; w++) v[w] = red[w * n + i];
#pragma unroll
    for (int w = 1; w < kRowWarps; w++) v[0] = __fadd_rn(v[0], v[w]);
    red[i] = v[0];
  }
  __syncthreads();
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

// y[m, n]: two CTAs of eight warps per SM, of which one computes while the
// other adds.  Each CTA, or cluster where there are few weight rows, takes a
// run of weight rows n, cut at multiples of eight so that all have about the
// same number, and goes through it 16 at a time; a warp goes through 256
// columns of them at a time, and the next tiles' bytes are under way while a
// tile's sums are added.  NT * 8 columns of the mma hold rows x parts; their x
// comes from L1 and L2, AHEAD times 64 columns before it is used (32 rows x
// 8192^2: 34 us with one and 46 us with two, which spills; 8 rows 20.8 us with
// two, 22.0 with one).  One CTA of 16 warps and 32 weight rows that share x
// took as long for 8 rows and 7.1 instead of 6.6 us for one row x 4096^2.
template <int NT>
struct Forward {
  static constexpr bool TABLES = NT == 1;
  static constexpr int AHEAD = NT <= 2 ? 2 : 1;
  static constexpr int DEPTH = NT == 1 ? 2 : 3;      // tiles in a warp's ring
  static constexpr int SUMS = kTileR * (NT * 8 + 1);  // [weight row][column], an odd pitch
};
template <int KIND, int DT, int NT>
__global__ void __launch_bounds__(kRowThreads, 2) rows_forward_kernel(const RowArgs a) {
  using W = W4<KIND>;
  using S = Forward<NT>;
  using R = Ring<KIND, 256, kTileR>;
  constexpr int P = bf16_parts(DT), C = NT * 8, D = S::DEPTH;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const ring = sm + kTableBytes<S::TABLES> + warp * D * R::BYTES;
  float* const red = reinterpret_cast<float*>(sm + kTableBytes<S::TABLES> + kRowWarps * D * R::BYTES);
  const int in = (int)a.in, out = (int)a.out, steps = (in + 255) / 256, stride = kRowWarps << a.cluster;
  const int me = (int)cluster_rank() * kRowWarps + warp;
  const int mine = (steps - me + stride - 1) >> (a.cluster + 3);  // this warp's steps of a piece (me < stride)
  const int run = blockIdx.x >> a.cluster;
  const int first = 8 * (run * a.per + min(run, a.extra)), last = min(out, first + 8 * (a.per + (run < a.extra)));
  const uint32_t q0 = (uint32_t)reinterpret_cast<uintptr_t>(a.q), row_bytes = (uint32_t)(a.in / W::BE * W::SB);
  constexpr uint32_t STEP = 256 / W::BE * W::SB;
  // what is fetched next: step fs (of `mine`) of the rows from fr
  uintptr_t from = R::place(a, first, lane);
  int fr = first, fs = 0, slot = 0;
  const auto fetch = [&](int to) {
    const int s = me + fs * stride;
    if (fs < mine && fr < last)
      R::fetch(a, ring + to * R::BYTES, from, fr, min(last - fr, kTileR), s * 256, s * STEP, lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++fs >= mine) fs = 0, fr += kTileR, from += (uint64_t)row_bytes * kTileR;
  };
#pragma unroll 1
  for (int i = 0; i < D - 1; i++) fetch(i);
  make_tables<KIND, S::TABLES>(sm);
  const uint32_t lane4 = lane * 4, at0 = kTableBytes<S::TABLES> + warp * D * R::BYTES + g * R::PITCH + 16 * t / W::BE * W::SB;
  const uint32_t half = 16 * t % W::BE / 2;  // this lane's 16 of every 64 columns: a block, or half a block of 32
  const float scale = out_scale(a.o);
  Column<DT> cols[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) cols[n].set(a, n * 8 + g);
  // the columns' rows, AHEAD times 64 columns (zeros behind the rows' end)
  uint32_t x[S::AHEAD][NT][8];
  const auto load_x = [&](int k, uint32_t (*o)[8]) {
    const bool all = a.wide && k + 16 <= in;
#pragma unroll
    for (int n = 0; n < NT; n++) cols[n].load16(k, in, all, o[n]);
  };
#pragma unroll
  for (int h = 0; h < S::AHEAD; h++) load_x(me * 256 + 16 * t + 64 * h, x[h]);
  __syncthreads();
#pragma unroll 1
  for (int r0 = first; r0 < last; r0 += kTileR) {
    float acc[NT][4] = {};
#pragma unroll 1
    for (int i = 0; i < mine; i++) {
      const int s = me + i * stride, k0 = s * 256 + 16 * t;
      const int next = i + 1 < mine ? k0 + stride * 256 : me * 256 + 16 * t;  // where the step after this one begins
      __syncwarp();  // all lanes are done with the stage that is filled next
      fetch(slot == 0 ? D - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
      __syncwarp();
      const uint32_t sk = q0 + (uint32_t)(r0 + g) * row_bytes + (uint32_t)s * STEP;
      const uint32_t off = at0 + slot * R::BYTES;
      slot = slot + 1 == D ? 0 : slot + 1;
      // 64 columns are 34 or 36 bytes, 128 a multiple of four: two places a row
      constexpr uint32_t RUN = 64 / W::BE * W::SB;
      const uint32_t p0 = off + (sk & 15u), p1 = off + 8 * R::PITCH + ((sk + 8 * row_bytes) & 15u);
      const At16 e0[2] = {at16(p0, half), at16(p0 + RUN, half)}, e1[2] = {at16(p1, half), at16(p1 + RUN, half)};
      float part[NT][4] = {};  // 16 mma (a tensor core cuts low bits off)
#pragma unroll 1
      for (int b = 0; b < 4; b += S::AHEAD)
#pragma unroll
        for (int h = 0; h < S::AHEAD; h++) {
          const int run = b + h;
          uint32_t w0[2], w1[2], f0, f1, o0[8], o1[8];
          if (S::AHEAD == 1) {
            load16<KIND, S::TABLES>(sm, at16(p0 + RUN * run, half), 0, lane4, w0, f0);
            load16<KIND, S::TABLES>(sm, at16(p1 + RUN * run, half), 0, lane4, w1, f1);
          } else {
            load16<KIND, S::TABLES>(sm, e0[h & 1], RUN * (run - (h & 1)), lane4, w0, f0);
            load16<KIND, S::TABLES>(sm, e1[h & 1], RUN * (run - (h & 1)), lane4, w1, f1);
          }
          decode16<KIND, S::TABLES>(sm, lane4, w0[0], w0[1], f0, o0);
          decode16<KIND, S::TABLES>(sm, lane4, w1[0], w1[1], f1, o1);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 8; j += 2)
              mma16816(part[n], o0[j], o1[j], o0[j + 1], o1[j + 1], x[h][n][j], x[h][n][j + 1]);
          load_x(run + S::AHEAD < 4 ? k0 + 64 * (run + S::AHEAD) : next + 64 * (run + S::AHEAD - 4), x[h]);
        }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[n][j] = __fadd_rn(acc[n][j], part[n][j]);
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float* const d = red + warp * S::SUMS + g * (C + 1) + n * 8 + 2 * t;
      d[0] = acc[n][0], d[1] = acc[n][1];
      d[8 * (C + 1)] = acc[n][2], d[8 * (C + 1) + 1] = acc[n][3];
    }
    add_and_store(
        red, S::SUMS, kTileR * a.rows, P, 1, [&](int o) { return o % kTileR * (C + 1) + o / kTileR * P; },
        [&](int o, float v) {
          if (o % kTileR < last - r0) finish(a.o, scale, o / kTileR, (int64_t)r0 + o % kTileR, v);
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
  using R = Ring<KIND, kDK, kTileR>;
  constexpr int P = bf16_parts(DT), C = NT * 8;
  extern __shared__ __align__(16) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t k0 = (int64_t)(blockIdx.x / cluster_size()) * kDK;
  const int64_t steps = (a.out + kTileR - 1) / kTileR, stride = (int64_t)kRowWarps * cluster_size();
  uint8_t* const ring = sm + kTableBytes<true> + warp * kDepth * R::BYTES;
  // A warp's sums, [column][17 floats per 16 k].  Where it has more than 32
  // steps they have a place of their own and take the accumulators in every
  // 32 mma (a tensor core cuts low bits off); else they lie where the ring was.
  float* const sums = reinterpret_cast<float*>(sm + (a.keep ? kTableBytes<true> + kRowWarps * kDepth * R::BYTES : 0));
  int64_t ahead = (int64_t)cluster_rank() * kRowWarps + warp;
  uint32_t y[NT][2];  // of the next step
  Column<DT> cols[NT];
#pragma unroll
  for (int n = 0; n < NT; n++) {
    cols[n].set(a, n * 8 + g);
    cols[n].load(ahead * kTileR + 4 * t, a.out, a.wide, y[n]);
  }
  make_tables<KIND, true>(sm);
  __syncthreads();
  const uint32_t q0 = (uint32_t)reinterpret_cast<uintptr_t>(a.q), row_bytes = (uint32_t)(a.in / W::BE * W::SB);
  const uint32_t sk = q0 + (uint32_t)(k0 / W::BE) * W::SB;
  // this lane's 16 columns: a block, or half a block of 32
  const uint32_t at0 = kTableBytes<true> + warp * kDepth * R::BYTES + 16 * g / W::BE * W::SB, half = 16 * g % W::BE / 2;
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
      if (ahead < steps) {
        const int r0 = (int)ahead * kTileR;
        R::fetch(a, ring + slot * R::BYTES, R::place(a, r0, lane), r0, min(kTileR, (int)a.out - r0), (int)k0,
                 (int)k0 / W::BE * W::SB, lane);
      }
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
        load16<KIND, true>(sm, at16(block, half), 0, lane * 4, w, f);
        if (n0 + r >= a.out) w[0] = w[1] = f = 0;  // behind the last row: whatever the stage held
        decode16<KIND, true>(sm, lane * 4, w[0], w[1], f, o[r]);
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
  add_and_store(
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

// CTAs that share a tile: `ctas` are launched at most, and fewer tiles than
// that are shared while every CTA still has a step for its warps
int cluster_for(int64_t tiles, int64_t steps, int ctas) {
  int cluster = 1;
  while (cluster < 8 && tiles * cluster * 2 <= ctas && cluster < steps) cluster *= 2;
  return cluster;
}

// smem: this launch's shared memory, most: the most of any launch of the kernel
template <void (*kernel)(const RowArgs)>
cudaError_t launch_rows(const RowArgs& a, int64_t tiles, int cluster, int smem, int most, cudaStream_t st) {
  static PerDevice set;
  if (const cudaError_t e = allow_shared(set, (const void*)kernel, most)) return e;
  if (cluster == 1) {
    kernel<<<(unsigned)tiles, kRowThreads, smem, st>>>(a);
    return cudaGetLastError();
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
cudaError_t launch_one(const LinearArgs& l, RowArgs a, int sms, cudaStream_t st) {
  if (l.op == LIN_FORWARD) {
    using S = Forward<NT>;
    const int64_t units = (a.out + 7) / 8;
    const int cluster = cluster_for(units, (a.in + 256 * kRowWarps - 1) / (256 * kRowWarps), 2 * sms);
    const int64_t runs = std::min<int64_t>(units, 2 * sms / cluster);
    while (1 << a.cluster < cluster) a.cluster++;
    a.per = (int)(units / runs), a.extra = (int)(units % runs);
    constexpr int smem = kTableBytes<S::TABLES> + kRowWarps * (S::DEPTH * Ring<KIND, 256, kTileR>::BYTES + S::SUMS * 4);
    return launch_rows<rows_forward_kernel<KIND, DT, NT>>(a, runs, cluster, smem, smem, st);
  }
  if constexpr (NT <= 2) {
    constexpr int ring = kTableBytes<true> + kRowWarps * kDepth * Ring<KIND, kDK, kTileR>::BYTES, sums = kRowWarps * NT * 8 * kRedPitch * 4;
    const int64_t tiles = (a.in + kDK - 1) / kDK, steps = (a.out + kTileR - 1) / kTileR;
    const int cluster = cluster_for(tiles, (steps + kRowWarps - 1) / kRowWarps, 2 * sms);
    a.keep = steps > 32 * (int64_t)kRowWarps * cluster;
    return launch_rows<rows_dgrad_kernel<KIND, DT, NT>>(a, tiles, cluster, a.keep ? ring + sums : std::max(ring, sums),
                                                        ring + sums, st);
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

cudaError_t rows_shared_limit(int* bytes) {
  cudaFuncAttributes f;
  const cudaError_t e = cudaFuncGetAttributes(&f, rows_dgrad_kernel<Q_MXFP4, DT_BF16, 1>);
  *bytes = e == cudaSuccess ? f.maxDynamicSharedSizeBytes : 0;
  return e;
}

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
  a.keep = a.cluster = a.per = a.extra = 0;
  a.wide = (reinterpret_cast<uintptr_t>(l.a) & 15u) == 0 && (l.rows == 1 || (l.lda * (l.a_dtype == DT_F32 ? 4 : 2)) % 16 == 0);
  if (l.kind == Q_MXFP4) return launch_dt<Q_MXFP4>(l, a, sms, st);
  if (l.kind == Q_MXFP4_OCP) return launch_dt<Q_MXFP4_OCP>(l, a, sms, st);
  return launch_dt<Q_NVFP4>(l, a, sms, st);
}

}  // namespace ody
