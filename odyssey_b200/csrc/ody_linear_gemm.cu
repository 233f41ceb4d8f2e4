// ody_linear_gemm.cu -- many rows: the quantised operand is brought to
// bfloat16 (exactly) once in the workspace, the other one too unless it can
// be read where it lies, and a tcgen05 kernel multiplies them.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "ody_linear_dev.cuh"
#include "ody_linear_gemm.h"

namespace ody {

// The kernels of one call follow each other as programmatic dependents: each
// is set up while the one before it still runs, and waits (previous_done)
// before it touches what that one wrote.  Every one of them waits, so that
// the end of the last means the end of all.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void previous_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------------------
// Bringing operands to bfloat16: one launch, whose first CTAs take the
// quantised operand and whose others, if any, take x or dy.  (A launch each
// cost 3 us more on the host, and on the GPU the smaller one's time.)
// ---------------------------------------------------------------------------
struct PrepareArgs {
  const uint8_t* q;
  const uint8_t* scales;  // wgrad
  int64_t qrows, qcols, qp;
  uint16_t* q16;  // [qrows, qp]
  unsigned q_ctas;
  const void* x;
  int64_t rows, cols, ld, pitch, plane;
  uint16_t* x16;  // planes of [rows, pitch]
  int wide;       // x's rows are 16-byte aligned
};

// Rows of whole blocks: the weight is one flat run of blocks, so are its
// bfloat16 values.  A tile of 8192 elements is 4608 or 4352 bytes, copied to
// shared memory with 16-byte loads; every thread then decodes eight elements
// four times, so that neighbouring threads write neighbouring 16 bytes.
constexpr int kUnpackTile = 8192;
template <int KIND>
__device__ __forceinline__ void unpack_w4_flat(const PrepareArgs& p) {
  using W = W4<KIND>;
  constexpr int TB = kUnpackTile / W::BE * W::SB;
  __shared__ __align__(16) uint8_t sm[TB + 32];
  const int64_t t = blockIdx.x, numel = p.qrows * p.qcols, b0 = t * TB, bytes = numel / W::BE * W::SB;
  const int n = (int)(bytes - b0 < TB ? bytes - b0 : TB);
  const uint8_t* src = p.q + b0;
  const int skew = (int)(reinterpret_cast<uintptr_t>(src) & 15u);
  // 16-byte words that lie wholly inside the tile, single bytes around them
  const int head = skew ? 16 - skew : 0;
  for (int i = threadIdx.x; i * 16 + head + 16 <= n; i += 256)
    *reinterpret_cast<uint4*>(sm + (skew ? 16 : 0) + i * 16) = __ldcs(reinterpret_cast<const uint4*>(src + head + i * 16));
  if ((int)threadIdx.x < head && (int)threadIdx.x < n) sm[skew + threadIdx.x] = src[threadIdx.x];
  const int rest = head + (n > head ? (n - head) / 16 * 16 : 0);
  if ((int)threadIdx.x < n - rest) sm[skew + rest + threadIdx.x] = src[rest + threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kUnpackTile / 2048; h++) {
    const int e = h * 2048 + threadIdx.x * 8;
    if (t * kUnpackTile + e >= numel) break;
    const int blk = skew + e / W::BE * W::SB, at = blk + (e % W::BE) / 2;
    const uint32_t* wp = reinterpret_cast<const uint32_t*>(sm) + (at >> 2);
    const uint32_t w = __funnelshift_r(wp[0], wp[1], 8 * (at & 3));
    const uint32_t sc = w4_scale_bf16x2<KIND>(sm[blk + W::SB - 1]);
    uint32_t o[4];
    w4_raw8<KIND>(w, o);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = mul_bf16x2(mul_bf16x2(o[i], kTwo126), sc);
    *reinterpret_cast<uint4*>(p.q16 + t * kUnpackTile + e) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// Any width: eight columns of a row per thread, the row padded to qp columns.
template <int KIND>
__device__ __forceinline__ void unpack_w4_rows(const PrepareArgs& p) {
  const int64_t n = p.qrows * (p.qp / 8), stride = (int64_t)p.q_ctas * 256;
  const bool blocks = p.qcols % 8 == 0;  // eight columns share a block
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += stride) {
    const int64_t r = t / (p.qp / 8), c = (t - r * (p.qp / 8)) * 8;
    EightQ<LIN_FORWARD, KIND> e;
    e.load(p.q, nullptr, p.qcols, r, c, (int)min((int64_t)8, p.qcols - c), blocks);
    e.store(reinterpret_cast<uint8_t*>(p.q16 + r * p.qp + c));
  }
}

// 8-bit activations: eight columns per thread, rows of whole groups.
template <int FMT>
__device__ __forceinline__ void unpack_a8(const PrepareArgs& p) {
  const int64_t t0 = (int64_t)blockIdx.x * 1024 + threadIdx.x, n8 = p.qrows * p.qp / 8;
  uint2 cs[4];
  uint32_t sbs[4];
#pragma unroll
  for (int h = 0; h < 4; h++) {
    const int64_t t = min(t0 + h * 256, n8 - 1);
    cs[h] = __ldcs(reinterpret_cast<const uint2*>(p.q) + t);
    sbs[h] = __ldg(p.scales + (t >> 2));
  }
#pragma unroll
  for (int h = 0; h < 4; h++) {
    const int64_t t = t0 + h * 256;
    if (t >= n8) return;
    float v[8];
    uint32_t o[4];
    a8_values8<FMT>(cs[h], sbs[h], v);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
    reinterpret_cast<uint4*>(p.q16)[t] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// x or dy as bf16_parts(DT) planes of [rows, pitch] bfloat16, zeros behind cols.
template <int DT>
__device__ __forceinline__ void pack_planes(const PrepareArgs& p) {
  constexpr int P = bf16_parts(DT);
  const int64_t n = p.rows * (p.pitch / 8), stride = (int64_t)(gridDim.x - p.q_ctas) * 256;
  for (int64_t t = (int64_t)(blockIdx.x - p.q_ctas) * 256 + threadIdx.x; t < n; t += stride) {
    const int64_t r = t / (p.pitch / 8), c = (t - r * (p.pitch / 8)) * 8, at = r * p.ld + c;
    uint16_t h[8][3];
    if (DT == DT_F32 && p.wide && c + 8 <= p.cols) {
      const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + at);
      const float4 a = __ldg(s), b = __ldg(s + 1);
      const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; i++) split_bf16(v[i], h[i][0], h[i][1], h[i][2]);
    } else if (DT != DT_F32 && p.wide && c + 8 <= p.cols) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + at));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint16_t b = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        if (DT == DT_BF16)
          h[i][0] = b;
        else
          split_bf16(f16_bits_to_f32(b), h[i][0], h[i][1], h[i][2]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        split_bf16(c + i < p.cols ? load_elem(p.x, DT, at + i) : 0.0f, h[i][0], h[i][1], h[i][2]);
    }
#pragma unroll
    for (int k = 0; k < P; k++)
      *reinterpret_cast<uint4*>(p.x16 + k * p.plane + r * p.pitch + c) =
          make_uint4(h[0][k] | (uint32_t)h[1][k] << 16, h[2][k] | (uint32_t)h[3][k] << 16,
                     h[4][k] | (uint32_t)h[5][k] << 16, h[6][k] | (uint32_t)h[7][k] << 16);
  }
}

enum : int { Q_FLAT, Q_ROWS, Q_ACT8 };  // how the quantised operand lies
template <int HOW, int KIND, int DT>
__global__ void __launch_bounds__(256) prepare_kernel(const PrepareArgs p) {
  let_next_start();
  if (blockIdx.x >= p.q_ctas)
    pack_planes<DT>(p);
  else if constexpr (HOW == Q_FLAT)
    unpack_w4_flat<KIND>(p);
  else if constexpr (HOW == Q_ROWS)
    unpack_w4_rows<KIND>(p);
  else
    unpack_a8<KIND>(p);
}

// ---------------------------------------------------------------------------
// The product: C[m, n] = sum over planes and r of A_p(m, r) B(n, r)
//
// Persistent CTA pairs, one CTA per SM, 256 x 256 results per pair.  In each
// CTA warp 0 copies its 128 x 64 of A and its 128 x 64 of B per step by TMA
// (128-byte swizzle) through six stages; the first CTA's warp 1 issues four
// tcgen05.mma.cta_group::2 (256 x 256 x 16) per step, which read both CTAs'
// halves, into one of two TMEM accumulators; warps 4 to 11 of each CTA take
// its 128 finished rows out.  The pair halves what every SM loads: one CTA
// alone with 128 x 256 results needs 48 KB per 512 cycles of MMA from L2 and
// reached 0.54 of the pair's rate.
//
// An operand whose rows are the reduction's (dgrad's W, both of wgrad's) is
// copied the same way, 64 columns at a time, and multiplied as "MN-major".
//
// The tensor core cuts off the low bits of what it adds, so a long sum in one
// accumulator drifts: over 8192 products to a relative 6e-6 (measured), where
// rounded float32 sums are 2e-7 off.  Every 512 products (1024 where the
// result is rounded to 16 bits) the accumulator is therefore taken to
// registers and added there with rounding (3e-7 and 6e-7), while the tensor
// core fills the other one.
//
// Tiles rarely fill a whole number of rounds of the 74 pairs.  Those that do
// not are dealt out by steps instead, evenly to all pairs, before the whole
// ones; the pieces of a shared tile are added in their order by gemm_join.
// (Adding them here, in whichever warp finished last, took 10 to 40 us: eight
// warps per SM cannot keep enough loads in flight.)
//
// A finished block of 32 columns goes through a 32 x 32 transpose in shared
// memory so that a row's columns leave together; the loop over the blocks is
// kept rolled (the accumulator moves down by 32 registers instead), because
// straight-line code is read cold by every launch and cost 11,000 cycles a
// block.
// ---------------------------------------------------------------------------
constexpr int kBM = 256, kBN = 256, kBK = 64, kStages = 6;
constexpr int kHalf = 128;                                   // rows of A and of B in each CTA
constexpr int kHalfBytes = kHalf * kBK * 2, kStageBytes = 2 * kHalfBytes;
constexpr int kEpiBytes = 8 * 32 * 32 * 4;                   // the epilogue's 32 x 32 transposes
constexpr int kGemmSmem = kStages * kStageBytes + kEpiBytes + 1024;
constexpr int kGemmThreads = 384;
// bound on every wait, in cycles of the SM's counter: 2 s at 2 GHz
constexpr long long kWaitCycles = 4000000000ll;

// set when a bounded wait ran out; read and cleared by gemm_wait_error
__device__ unsigned g_gemm_err;

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// false: the wait ran out, or another warp's did
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                                          long long limit = kWaitCycles) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort) return false;
    if (clock64() - t0 > limit) {
      *abort = 1;
      atomicExch(&g_gemm_err, 1u);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {  // the same place in a CTA of the pair
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// a box into this CTA's memory; its bytes count on a barrier of either CTA
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// arrives at the barrier in both CTAs when the MMAs issued so far are done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   bar),
               "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Shared-memory descriptor of a 128-byte-swizzled operand: K-major, rows of
// 64 k at 128 bytes, eight rows every 1024 bytes; MN-major, the same rows are
// k and hold 64 columns, the next 64 columns lie kBK * 128 bytes on.
template <bool MN>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  const uint64_t lbo = MN ? (kBK * 128) >> 4 : 1, sbo = 1024 >> 4;
  return (uint64_t)((addr & 0x3ffff) >> 4) | lbo << 16 | sbo << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

struct GemmArgs {
  LinearOut o;
  int64_t M, N;
  int tiles_m, tiles_n;
  int steps;          // of 64 of the reduction, per plane
  int total;          // steps * planes: of one tile
  int chunk;          // steps in one accumulator
  // The first `shared` tiles' steps are dealt out evenly, `deal` to each pair
  // of SMs whether or not tiles end there; the other tiles, a multiple of the
  // number of pairs, go to one pair each.
  int shared;
  int deal;
  float* partial;     // two slots of 256 x 256 per pair: its first and its last piece of a tile, in rows
};

// tile t's place: bands of eight row tiles, so that CTAs running at once share
// rows of A and columns of B in L2
__device__ __forceinline__ void tile_at(const GemmArgs& g, int t, int& tm, int& tn) {
  const int band = 8 * g.tiles_n, b = t / band, first = b * 8;
  const int h = min(8, g.tiles_m - first), in = t - b * band;
  tm = first + in % h;
  tn = in / h;
}

// what a pair of SMs works off, piece by piece
struct Pieces {
  int64_t pos, end;  // of the shared tiles' steps
  int next;          // whole tile
  int tile, s0, s1;
  __device__ __forceinline__ Pieces(const GemmArgs& g, int pair) {
    const int64_t all = (int64_t)g.shared * g.total;
    pos = min((int64_t)pair * g.deal, all);
    end = min(pos + g.deal, all);
    next = g.shared + pair;
  }
  __device__ __forceinline__ bool get(const GemmArgs& g, int pairs) {
    if (pos < end) {
      tile = (int)(pos / g.total);
      s0 = (int)(pos - (int64_t)tile * g.total);
      s1 = (int)min((int64_t)g.total, s0 + (end - pos));
      pos += s1 - s0;
      return true;
    }
    if (next >= g.tiles_m * g.tiles_n) return false;
    tile = next, s0 = 0, s1 = g.total;
    next += pairs;
    return true;
  }
};

// A warp's 32 x 32 results, one row per lane, turned in shared memory (rows of
// 128 bytes, their 16-byte pieces exchanged by the row's number so that
// neither side meets a bank twice) and stored at c, rows of ld.
__device__ __forceinline__ float4* piece_of(float* buf, int row, int piece) {
  return reinterpret_cast<float4*>(buf) + row * 8 + (piece ^ (row & 7));
}
template <int DT>
__device__ __forceinline__ void store_block(float* buf, void* c, const void* add, int64_t ld, float scale, int rows, int cols,
                                            int lane) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const auto bits = [](float v) { return DT == DT_F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v); };
  if (cols >= 32 && ((reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(add) | (uintptr_t)(ld * ES)) &
                     (uintptr_t)(4 * ES - 1)) == 0) {
    // four columns per lane, four rows at a time
    const int64_t at = ((lane >> 3) * ld + (lane & 7) * 4) * ES;
    uint8_t* d = reinterpret_cast<uint8_t*>(c) + at;
    const uint8_t* e = reinterpret_cast<const uint8_t*>(add) + at;
#pragma unroll 2
    for (int r = lane >> 3; r < rows; r += 4, d += 4 * ld * ES, e += 4 * ld * ES) {
      float4 v = *piece_of(buf, r, lane & 7);
      v.x = __fmul_rn(v.x, scale), v.y = __fmul_rn(v.y, scale), v.z = __fmul_rn(v.z, scale), v.w = __fmul_rn(v.w, scale);
      if (add) {
        float w[4];
        if constexpr (DT == DT_F32) {
          const float4 f = *reinterpret_cast<const float4*>(e);
          w[0] = f.x, w[1] = f.y, w[2] = f.z, w[3] = f.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(e);
          const uint16_t h[4] = {(uint16_t)u.x, (uint16_t)(u.x >> 16), (uint16_t)u.y, (uint16_t)(u.y >> 16)};
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = DT == DT_F16 ? f16_bits_to_f32(h[k]) : bf16_bits_to_f32(h[k]);
        }
        v.x = __fadd_rn(v.x, w[0]), v.y = __fadd_rn(v.y, w[1]), v.z = __fadd_rn(v.z, w[2]), v.w = __fadd_rn(v.w, w[3]);
      }
      if constexpr (DT == DT_F32)
        *reinterpret_cast<float4*>(d) = v;
      else
        *reinterpret_cast<uint2*>(d) =
            make_uint2(bits(v.x) | (uint32_t)bits(v.y) << 16, bits(v.z) | (uint32_t)bits(v.w) << 16);
    }
  } else if (lane < cols) {
    // any alignment: a column per lane; what is added comes four rows at a time
    uint8_t* d = reinterpret_cast<uint8_t*>(c) + lane * ES;
    const uint8_t* e = reinterpret_cast<const uint8_t*>(add) + lane * ES;
    const int64_t step = ld * ES;
#pragma unroll 1
    for (int r = 0; r < rows; r += 4, d += 4 * step, e += 4 * step) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        v[k] = __fmul_rn(reinterpret_cast<const float*>(piece_of(buf, r + k, lane >> 2))[lane & 3], scale);
      if (add) {
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = r + k < rows ? load_elem(e + k * step, DT, 0) : 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = __fadd_rn(v[k], w[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (r + k < rows) {
          if constexpr (DT == DT_F32)
            *reinterpret_cast<float*>(d + k * step) = v[k];
          else
            *reinterpret_cast<uint16_t*>(d + k * step) = bits(v[k]);
        }
    }
  }
}

// tcgen05.ld of 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t v[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

template <bool AMN, bool BMN, int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const GemmArgs g) {
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const uint32_t smem = (srow(dyn) + 1023u) & ~1023u;
  const uint32_t full = srow(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16,
                 drain = tempty + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  volatile int* abort = &abort_flag;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; i++) mbar_init(tfull + 8 * i, 1), mbar_init(tempty + 8 * i, 16);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(srow(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_barrier();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;
  let_next_start();
  previous_done();
  // registers: 4 warps x 32 x 64 + 8 x 32 x 216 of the launch's 384 x 168
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 0 && lane == 0) {
    int it = 0;
    const uint32_t lead = in_cta(full, 0);
    bool ok = true;
    Pieces w(g, pair);
    while (ok && !*abort && w.get(g, pairs)) {
      int tm, tn;
      tile_at(g, w.tile, tm, tn);
      const int am = tm * kBM + rank * kHalf, bn = tn * kBN + rank * kHalf;
      for (int s = w.s0; s < w.s1; s++, it++) {
        const int st = it % kStages;
        if (it >= kStages && !(ok = mbar_wait(empty + 8 * st, (it / kStages - 1) & 1, abort))) break;
        const uint32_t a = smem + st * kStageBytes, b = a + kHalfBytes, bar = lead + 8 * st;
        const int p = s / g.steps, r = (s - p * g.steps) * kBK;
        if (rank == 0) mbar_expect(full + 8 * st, 2 * kStageBytes);
        if (AMN) {
#pragma unroll
          for (int i = 0; i < kHalf / 64; i++) tma_load3(a + i * kBK * 128, &ma, bar, am + i * 64, r, p);
        } else {
          tma_load3(a, &ma, bar, r, am, p);
        }
        if (BMN) {
#pragma unroll
          for (int i = 0; i < kHalf / 64; i++) tma_load3(b + i * kBK * 128, &mb, bar, bn + i * 64, r, 0);
        } else {
          tma_load3(b, &mb, bar, r, bn, 0);
        }
      }
    }
    if (*abort && rank == 0) {  // no copy may still be in flight when the CTAs' memory goes
      for (int i = it > kStages ? it - kStages : 0; i < it; i++) {
        const long long t0 = clock64();
        while (!mbar_try(full + 8 * (i % kStages), (i / kStages) & 1) && clock64() - t0 < kWaitCycles) {
        }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // D float32, A and B bfloat16, majors, N, M
    constexpr uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)AMN << 15 | (uint32_t)BMN << 16 |
                               (uint32_t)(kBN >> 3) << 17 | (uint32_t)(kBM >> 4) << 24;
    int it = 0, chunk = 0;
    bool ok = true;
    Pieces w(g, pair);
    while (ok && !*abort && w.get(g, pairs)) {
      for (int c = w.s0; c < w.s1 && ok; c += g.chunk, chunk++) {
        const int buf = chunk & 1;
        if (chunk >= 2 && !(ok = mbar_wait(tempty + 8 * buf, (chunk / 2 - 1) & 1, abort))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int ce = min(c + g.chunk, w.s1);
        for (int s = c; s < ce; s++, it++) {
          const int st = it % kStages;
          if (!(ok = mbar_wait(full + 8 * st, (it / kStages) & 1, abort))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a = smem + st * kStageBytes, b = a + kHalfBytes;
#pragma unroll
          for (int k = 0; k < kBK / 16; k++)
            mma_f16(tmem + buf * kBN, smem_desc<AMN>(a + k * (AMN ? 2048 : 32)), smem_desc<BMN>(b + k * (BMN ? 2048 : 32)),
                    idesc, s > c || k > 0);
          mma_commit(empty + 8 * st);
        }
        if (ok) mma_commit(tfull + 8 * buf);
      }
    }
    if (*abort) {  // nor an MMA
      mma_commit(drain);
      const long long t0 = clock64();
      while (!mbar_try(drain, 0) && clock64() - t0 < kWaitCycles) {
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + half * (kBN / 2);
    const uint32_t done = in_cta(tempty, 0);
    // a warp goes on, or stops after a wait that ran out, as one
    const auto together = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
    float* buf32 = reinterpret_cast<float*>(dyn + (smem - srow(dyn)) + kStages * kStageBytes) + (warp - 4) * 32 * 32;
    const float scale = out_scale(g.o);
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    int chunk = 0;
    bool ok = true;
    Pieces w(g, pair);
    while (ok && together(!*abort) && w.get(g, pairs)) {
      int tm, tn;
      tile_at(g, w.tile, tm, tn);
      float acc[kBN / 2];
#pragma unroll
      for (int i = 0; i < kBN / 2; i++) acc[i] = 0.0f;
      for (int c = w.s0; c < w.s1; c += g.chunk, chunk++) {
        const int buf = chunk & 1;
        if (!(ok = together(mbar_wait(tfull + 8 * buf, (chunk / 2) & 1, abort)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // 32 columns are added while the next 32 are on their way
        uint32_t v[2][32];
        tmem_load32(taddr + buf * kBN, v[0]);
#pragma unroll
        for (int j = 0; j < kBN / 2; j += 32) {
          tmem_wait();
          if (j + 32 < kBN / 2) tmem_load32(taddr + buf * kBN + j + 32, v[(j / 32 + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 32; i++) acc[j + i] = __fadd_rn(acc[j + i], __uint_as_float(v[(j / 32) & 1][i]));
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(done + 8 * buf);
      }
      if (!ok) break;
      const int64_t m0 = (int64_t)tm * kBM + rank * kHalf + quarter * 32, n0 = (int64_t)tn * kBN + half * (kBN / 2);
      if (m0 >= g.M || n0 >= g.N) continue;
      const bool part = w.s1 - w.s0 < g.total;  // of a shared tile
      const int rows = (int)min((int64_t)32, g.M - m0);
      uint8_t* c;
      const uint8_t* add = nullptr;
      if (part) {
        c = reinterpret_cast<uint8_t*>(g.partial + (int64_t)(2 * pair + (w.s0 == 0)) * kBM * kBN +
                                       (rank * kHalf + quarter * 32) * kBN + half * (kBN / 2));
      } else {
        const int64_t at = (m0 * g.o.ld + n0) * ES;
        c = reinterpret_cast<uint8_t*>(g.o.c) + at;
        if (g.o.add) add = reinterpret_cast<const uint8_t*>(g.o.add) + at;
      }
#pragma unroll 1
      for (int cols = (int)min((int64_t)(kBN / 2), g.N - n0); cols > 0; cols -= 32) {
#pragma unroll
        for (int i = 0; i < 8; i++)
          *piece_of(buf32, lane, i) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
#pragma unroll
        for (int i = 0; i < kBN / 2 - 32; i++) acc[i] = acc[i + 32];
        __syncwarp();
        if (part) {
          store_block<DT_F32>(buf32, c, nullptr, kBN, 1.0f, rows, 32, lane);  // whole: its place is 256 wide
          c += 32 * 4;
        } else {
          store_block<DT>(buf32, c, add, g.o.ld, scale, rows, cols, lane);
          c += 32 * ES;
          if (add) add += 32 * ES;
        }
        __syncwarp();
      }
    }
  }
  __syncthreads();
  if (*abort && warp == 0) {  // what the other CTA's copies still do ends in this time
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {
    }
  }
  __syncwarp();
  cluster_barrier();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The shared tiles' results: their pieces added in the order of the steps.  64
// threads per row with four columns each, eight rows per CTA.
__global__ void __launch_bounds__(256) gemm_join_kernel(const GemmArgs g) {
  previous_done();
  const int tile = blockIdx.x >> 5;
  int tm, tn;
  tile_at(g, tile, tm, tn);
  const int64_t t0 = (int64_t)tile * g.total;
  const int first = (int)(t0 / g.deal), last = (int)((t0 + g.total - 1) / g.deal);
  if (first == last) return;  // a whole tile
  const float scale = out_scale(g.o);
  const int c = (threadIdx.x & 63) * 4;
  const int64_t n = (int64_t)tn * kBN + c;
  if (n >= g.N) return;
  const int w = (int)min((int64_t)4, g.N - n);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = (blockIdx.x & 31) * 8 + h * 4 + (threadIdx.x >> 6);
    const int64_t m = (int64_t)tm * kBM + r;
    if (m >= g.M) return;
    const float* s = g.partial + r * kBN + c;
    float4 v = *reinterpret_cast<const float4*>(s + (int64_t)(2 * first + 1) * kBM * kBN);  // the tile's begin
#pragma unroll 4
    for (int q = first + 1; q <= last; q++) {
      const float4 f = *reinterpret_cast<const float4*>(s + (int64_t)(2 * q) * kBM * kBN);  // begins inside the tile
      v.x = __fadd_rn(v.x, f.x), v.y = __fadd_rn(v.y, f.y), v.z = __fadd_rn(v.z, f.z), v.w = __fadd_rn(v.w, f.w);
    }
    float x[4] = {v.x, v.y, v.z, v.w};
    const int es = g.o.dtype == DT_F32 ? 4 : 2;
    const int64_t at = m * g.o.ld + n;
    if (w == 4 && ((reinterpret_cast<uintptr_t>(g.o.c) | reinterpret_cast<uintptr_t>(g.o.add) | (uintptr_t)(g.o.ld * es)) &
                   (uintptr_t)(4 * es - 1)) == 0) {  // four results together
#pragma unroll
      for (int k = 0; k < 4; k++) x[k] = __fmul_rn(x[k], scale);
      if (es == 4) {
        if (g.o.add) {
          const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(g.o.add) + at);
          x[0] = __fadd_rn(x[0], f.x), x[1] = __fadd_rn(x[1], f.y), x[2] = __fadd_rn(x[2], f.z), x[3] = __fadd_rn(x[3], f.w);
        }
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(g.o.c) + at) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        const bool half = g.o.dtype == DT_F16;
        if (g.o.add) {
          const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(g.o.add) + at);
          const uint16_t f[4] = {(uint16_t)u.x, (uint16_t)(u.x >> 16), (uint16_t)u.y, (uint16_t)(u.y >> 16)};
#pragma unroll
          for (int k = 0; k < 4; k++) x[k] = __fadd_rn(x[k], half ? f16_bits_to_f32(f[k]) : bf16_bits_to_f32(f[k]));
        }
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = half ? f32_to_f16_bits(x[k]) : f32_to_bf16_bits(x[k]);
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(g.o.c) + at) = make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (k < w) finish(g.o, scale, m, n + k, x[k]);
    }
  }
}

// A wait for a barrier that nothing arrives at (the time-out path's test).
__global__ void wait_selftest_kernel(long long limit) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  abort_flag = 0;
  mbar_init(srow(&bar), 1);
  mbar_wait(srow(&bar), 0, &abort_flag, limit);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// planes x rows x cols of bfloat16, boxes of 64 columns and box_rows rows;
// what a box reads outside is zero
cudaError_t make_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t planes, int64_t pitch,
                     int64_t plane, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)plane * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// everything about a call that its shapes and types decide
struct Plan {
  int64_t M, N, R;              // the product's
  int64_t qrows, qcols, qp;     // the quantised operand as bfloat16, pitch qp
  int64_t arows, acols, ap;     // the other one, pitch of its planes ap
  int planes, steps, tiles_m, tiles_n, shared, deal;
  bool split;  // some tile is shared by several pairs
  int64_t q_off, a_off, p_off, bytes;
};

Plan make_plan(const LinearArgs& a, int sms) {
  Plan p;
  p.M = a.op == LIN_WGRAD ? a.out : a.rows;
  p.N = a.op == LIN_FORWARD ? a.out : a.in;
  p.R = a.op == LIN_FORWARD ? a.in : (a.op == LIN_DGRAD ? a.out : a.rows);
  p.qrows = a.op == LIN_WGRAD ? a.rows : a.out;
  p.qcols = a.in;
  p.qp = a.op == LIN_WGRAD ? up(a.in, kA8Group) : up(a.in, 8);
  p.arows = a.rows;
  p.acols = a.op == LIN_FORWARD ? a.in : a.out;
  p.ap = up(p.acols, 8);
  p.planes = bf16_parts(a.a_dtype);
  p.steps = (int)((p.R + kBK - 1) / kBK);
  p.tiles_m = (int)((p.M + kBM - 1) / kBM);
  p.tiles_n = (int)((p.N + kBN - 1) / kBN);
  // Tiles that do not fill a whole round of the pairs are dealt out by steps.
  // A tile is shared by about sqrt(total) / 2 pairs at most: a piece costs
  // about as long as four steps take.
  const int pairs = sms / 2;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, total = (int64_t)p.steps * p.planes;
  const int64_t shared = tiles % pairs;
  const int64_t most = std::max<int64_t>(1, (int64_t)(sqrt((double)total) / 2));
  int64_t deal = std::max((shared * total + pairs - 1) / pairs, (total + most - 1) / most);
  p.shared = (int)shared, p.deal = (int)std::max<int64_t>(deal, 1);
  p.split = shared > 0 && deal % total != 0;
  p.q_off = 0;
  p.a_off = up(p.q_off + p.qrows * p.qp * 2, 256);
  p.p_off = up(p.a_off + p.planes * p.arows * p.ap * 2, 256);
  p.bytes = p.p_off + (p.split ? (int64_t)pairs * 2 * kBM * kBN * 4 : 0);
  return p;
}

int grid_for(int64_t threads, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, (int64_t)sms * 8));
}

// a kernel that may be set up while the one before it in the stream runs
template <class... P, class... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

template <int HOW, int KIND>
cudaError_t prepare(const PrepareArgs& p, int dtype, int x_ctas, cudaStream_t st) {
  const unsigned grid = p.q_ctas + x_ctas;
  if (dtype == DT_F32)
    prepare_kernel<HOW, KIND, DT_F32><<<grid, 256, 0, st>>>(p);
  else if (dtype == DT_F16)
    prepare_kernel<HOW, KIND, DT_F16><<<grid, 256, 0, st>>>(p);
  else
    prepare_kernel<HOW, KIND, DT_BF16><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

template <int KIND>
cudaError_t prepare_w4(PrepareArgs& p, int dtype, int x_ctas, int sms, cudaStream_t st) {
  if (p.qcols % W4<KIND>::BE == 0) {
    p.q_ctas = (unsigned)((p.qrows * p.qcols + kUnpackTile - 1) / kUnpackTile);
    return prepare<Q_FLAT, KIND>(p, dtype, x_ctas, st);
  }
  p.q_ctas = grid_for(p.qrows * p.qp / 8, sms);
  return prepare<Q_ROWS, KIND>(p, dtype, x_ctas, st);
}

template <bool AMN, bool BMN, int DT>
cudaError_t run_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& g, int sms, cudaStream_t st) {
  static PerDevice set;
  if (const cudaError_t e = allow_shared(set, (const void*)gemm_kernel<AMN, BMN, DT>, kGemmSmem)) return e;
  // with whole tiles only, no more pairs than tiles
  const int64_t shares = ((int64_t)g.shared * g.total + g.deal - 1) / g.deal;
  const int64_t work = g.tiles_m * (int64_t)g.tiles_n > g.shared ? sms / 2 : shares;
  return launch_next(gemm_kernel<AMN, BMN, DT>, dim3((unsigned)std::min<int64_t>(work, sms / 2) * 2), kGemmThreads, kGemmSmem,
                     st, ma, mb, g);
}

}  // namespace

cudaError_t gemm_wait_error(cudaStream_t st, bool* ran_out) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_gemm_err, sizeof(v), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && v) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbolAsync(g_gemm_err, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  *ran_out = v != 0;
  return e;
}

cudaError_t launch_wait_selftest(long long cycles, cudaStream_t st) {
  wait_selftest_kernel<<<1, 1, 0, st>>>(cycles);
  return cudaGetLastError();
}

int64_t gemm_workspace(const LinearArgs& a, int sms) { return make_plan(a, sms).bytes; }

cudaError_t launch_gemm(const LinearArgs& a, void* ws, int sms, cudaStream_t st) {
  const Plan p = make_plan(a, sms);
  uint8_t* base = static_cast<uint8_t*>(ws);
  uint16_t* q16 = reinterpret_cast<uint16_t*>(base + p.q_off);
  PrepareArgs r{};
  r.q = a.q, r.scales = a.scales, r.qrows = p.qrows, r.qcols = p.qcols, r.qp = p.qp, r.q16 = q16;
  // bfloat16 rows that TMA can read are used where they lie
  const void* abase = a.a;
  int64_t apitch = a.lda, aplane = a.lda;  // one plane: its pitch is never used
  int x_ctas = 0;
  if (a.a_dtype != DT_BF16 || (reinterpret_cast<uintptr_t>(a.a) & 15u) || a.lda % 8) {
    const int64_t es = a.a_dtype == DT_F32 ? 4 : 2;
    apitch = p.ap, aplane = p.arows * p.ap;
    r.x = a.a, r.rows = p.arows, r.cols = p.acols, r.ld = a.lda, r.pitch = apitch, r.plane = aplane;
    r.x16 = reinterpret_cast<uint16_t*>(base + p.a_off);
    r.wide = (reinterpret_cast<uintptr_t>(a.a) & 15u) == 0 && (a.lda * es) % 16 == 0;
    x_ctas = grid_for(p.arows * p.ap / 8, sms);
    abase = r.x16;
  }
  cudaError_t e;
  if (a.op == LIN_WGRAD) {
    r.q_ctas = (unsigned)((p.qrows * p.qp / 8 + 1023) / 1024);
    e = a.kind == A8_E4M3 ? prepare<Q_ACT8, A8_E4M3>(r, a.a_dtype, x_ctas, st) : prepare<Q_ACT8, A8_E5M2>(r, a.a_dtype, x_ctas, st);
  } else if (a.kind == Q_MXFP4) {
    e = prepare_w4<Q_MXFP4>(r, a.a_dtype, x_ctas, sms, st);
  } else if (a.kind == Q_MXFP4_OCP) {
    e = prepare_w4<Q_MXFP4_OCP>(r, a.a_dtype, x_ctas, sms, st);
  } else {  // the tensor scale of ODY_Q_NVFP4_TENSOR is applied to the sums
    e = prepare_w4<Q_NVFP4>(r, a.a_dtype, x_ctas, sms, st);
  }
  if (e != cudaSuccess) return e;
  const bool amn = a.op == LIN_WGRAD, bmn = a.op != LIN_FORWARD;
  CUtensorMap ma, mb;
  if ((e = make_map(&ma, abase, p.acols, p.arows, p.planes, apitch, aplane, amn ? kBK : kHalf)) != cudaSuccess) return e;
  if ((e = make_map(&mb, q16, p.qcols, p.qrows, 1, p.qp, p.qp, bmn ? kBK : kHalf)) != cudaSuccess) return e;
  GemmArgs g;
  g.o = a.o;
  g.M = p.M, g.N = p.N;
  g.tiles_m = p.tiles_m, g.tiles_n = p.tiles_n;
  g.steps = p.steps, g.total = p.steps * p.planes, g.chunk = a.o.dtype == DT_F32 ? 8 : 16;
  g.shared = p.shared, g.deal = p.deal;
  g.partial = reinterpret_cast<float*>(base + p.p_off);
  const auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.op == LIN_FORWARD) return run_gemm<false, false, DT>(ma, mb, g, sms, st);
    return a.op == LIN_DGRAD ? run_gemm<false, true, DT>(ma, mb, g, sms, st) : run_gemm<true, true, DT>(ma, mb, g, sms, st);
  };
  e = a.o.dtype == DT_F32   ? run(std::integral_constant<int, DT_F32>())
      : a.o.dtype == DT_F16 ? run(std::integral_constant<int, DT_F16>())
                            : run(std::integral_constant<int, DT_BF16>());
  if (e != cudaSuccess || !p.split) return e;
  return launch_next(gemm_join_kernel, dim3((unsigned)p.shared * 32), 256, 0, st, g);
}

}  // namespace ody
