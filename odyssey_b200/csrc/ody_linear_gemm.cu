// ody_linear_gemm.cu -- many rows: the quantised operand is brought to
// bfloat16 (exactly) once in the workspace, the other one too unless it can
// be read where it lies, and a tcgen05 kernel multiplies them.
#include <cuda.h>

#include "ody_linear_dev.cuh"
#include "ody_linear_gemm.h"

namespace ody {

// ---------------------------------------------------------------------------
// Bringing operands to bfloat16
// ---------------------------------------------------------------------------

// Rows of whole blocks: the weight is one flat run of blocks, so are its
// bfloat16 values.  A tile of 2048 elements is 1152 or 1088 bytes, copied to
// shared memory with 16-byte loads; every thread decodes eight elements.
template <int KIND>
__global__ void __launch_bounds__(256) unpack_w4_flat_kernel(const uint8_t* __restrict__ q, int64_t numel,
                                                             uint16_t* __restrict__ out) {
  using W = W4<KIND>;
  constexpr int TB = 2048 / W::BE * W::SB;
  __shared__ __align__(16) uint8_t sm[TB + 16];
  const int64_t bytes = numel / W::BE * W::SB;
  const int64_t tiles = (numel + 2047) / 2048;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t b0 = t * TB;
    const int n = (int)(bytes - b0 < TB ? bytes - b0 : TB);
    const uint8_t* src = q + b0;
    const int skew = (int)(reinterpret_cast<uintptr_t>(src) & 15u);
    // 16-byte words that lie wholly inside the tile, single bytes around them
    const int head = skew ? 16 - skew : 0;
    for (int i = threadIdx.x; i * 16 + head + 16 <= n; i += 256)
      *reinterpret_cast<uint4*>(sm + (skew ? 16 : 0) + i * 16) =
          __ldg(reinterpret_cast<const uint4*>(src + head + i * 16));
    if ((int)threadIdx.x < head && (int)threadIdx.x < n) sm[skew + threadIdx.x] = src[threadIdx.x];
    const int rest = head + (n > head ? (n - head) / 16 * 16 : 0);
    if ((int)threadIdx.x < n - rest) sm[skew + rest + threadIdx.x] = src[rest + threadIdx.x];
    __syncthreads();
    const int e = threadIdx.x * 8;
    if (t * 2048 + e < numel) {
      const uint8_t* blk = sm + skew + e / W::BE * W::SB;
      const float sf = W::scale(blk[W::SB - 1]);
      const uint8_t* c = blk + (e % W::BE) / 2;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t b = c[i];
        // the product is exact in bfloat16, so its upper half is all of it
        o[i] = (__float_as_uint(W::value(b >> 4, sf)) >> 16) | (__float_as_uint(W::value(b & 15u, sf)) & 0xffff0000u);
      }
      *reinterpret_cast<uint4*>(out + t * 2048 + e) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
  }
}

// Any width: eight columns of a row per thread, the row padded to kp columns.
template <int KIND>
__global__ void __launch_bounds__(256) unpack_w4_rows_kernel(const uint8_t* __restrict__ q, int64_t rows, int64_t cols,
                                                             int64_t kp, uint16_t* __restrict__ out) {
  const int64_t n = rows * (kp / 8), stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += stride) {
    const int64_t r = t / (kp / 8), c = (t - r * (kp / 8)) * 8;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = c + 2 * i < cols ? W4<KIND>::at(q, r * cols + c + 2 * i) : 0.0f;
      const float b = c + 2 * i + 1 < cols ? W4<KIND>::at(q, r * cols + c + 2 * i + 1) : 0.0f;
      o[i] = (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u);
    }
    *reinterpret_cast<uint4*>(out + r * kp + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// 8-bit activations: sixteen columns per thread, rows of whole groups.
template <int FMT>
__global__ void __launch_bounds__(256) unpack_a8_kernel(const uint8_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales, int64_t n16,
                                                        uint16_t* __restrict__ out) {
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < n16; t += stride) {
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(codes) + t);
    const uint32_t sb = scales[t >> 1];
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t two = w[i >> 1] >> (16 * (i & 1));
      o[i] = (__float_as_uint(a8_value<FMT>(two & 255u, sb)) >> 16) |
             (__float_as_uint(a8_value<FMT>((two >> 8) & 255u, sb)) & 0xffff0000u);
    }
    uint4* d = reinterpret_cast<uint4*>(out) + 2 * t;
    d[0] = make_uint4(o[0], o[1], o[2], o[3]);
    d[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// x or dy as bf16_parts(DT) planes of [rows, cp] bfloat16, zeros behind cols.
template <int DT>
__global__ void __launch_bounds__(256) pack_planes_kernel(const void* __restrict__ x, int64_t rows, int64_t cols,
                                                          int64_t ldx, int64_t cp, int64_t plane, uint16_t* __restrict__ out,
                                                          int wide) {
  constexpr int P = bf16_parts(DT);
  const int64_t n = rows * (cp / 8), stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < n; t += stride) {
    const int64_t r = t / (cp / 8), c = (t - r * (cp / 8)) * 8, at = r * ldx + c;
    uint16_t h[8][3];
    if (DT == DT_F32 && wide && c + 8 <= cols) {
      const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + at);
      const float4 a = __ldg(s), b = __ldg(s + 1);
      const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; i++) split_bf16(v[i], h[i][0], h[i][1], h[i][2]);
    } else if (DT != DT_F32 && wide && c + 8 <= cols) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + at));
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
        split_bf16(c + i < cols ? load_elem(x, DT, at + i) : 0.0f, h[i][0], h[i][1], h[i][2]);
    }
#pragma unroll
    for (int p = 0; p < P; p++)
      *reinterpret_cast<uint4*>(out + p * plane + r * cp + c) =
          make_uint4(h[0][p] | (uint32_t)h[1][p] << 16, h[2][p] | (uint32_t)h[3][p] << 16,
                     h[4][p] | (uint32_t)h[5][p] << 16, h[6][p] | (uint32_t)h[7][p] << 16);
  }
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
// accumulator drifts; every 256 products the accumulator is therefore taken
// to registers and added there in float32 with rounding, while the tensor
// core fills the other one.
// ---------------------------------------------------------------------------
constexpr int kBM = 256, kBN = 256, kBK = 64, kStages = 6, kChunk64 = 4;
constexpr int kHalf = 128;                                   // rows of A and of B in each CTA
constexpr int kHalfBytes = kHalf * kBK * 2, kStageBytes = 2 * kHalfBytes;
constexpr int kStagePitch = 33;                              // floats; the epilogue's 32 x 32 transposes
constexpr int kEpiBytes = 8 * 32 * kStagePitch * 4;
constexpr int kGemmSmem = kStages * kStageBytes + kEpiBytes + 1024;
constexpr int kGemmThreads = 384;
constexpr unsigned long long kGemmWaitNs = 2000000000ull;  // bound on every wait (2 s)

// set when a bounded wait ran out; read and cleared by gemm_wait_error
__device__ unsigned g_gemm_err;

__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
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
                                          unsigned long long limit = kGemmWaitNs) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  while (!mbar_try(bar, parity)) {
    if (*abort) return false;
    if (now_ns() - t0 > limit) {
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
  int steps;         // of 64 of the reduction, per plane
  int planes;
  int splits;        // of planes * steps
  float* partial;    // splits > 1: [splits, M, N]
};

// tile t's place: bands of eight row tiles, so that CTAs running at once share
// rows of A and columns of B in L2
__device__ __forceinline__ void tile_at(const GemmArgs& g, int t, int& tm, int& tn) {
  const int band = 8 * g.tiles_n, b = t / band, first = b * 8;
  const int h = min(8, g.tiles_m - first), in = t - b * band;
  tm = first + in % h;
  tn = in / h;
}
__device__ __forceinline__ int split_at(const GemmArgs& g, int sp) {
  return (int)((int64_t)g.steps * g.planes * sp / g.splits);
}

// 32 columns of a warp's 32 rows out, through shared memory so that a row's
// columns leave together: with one thread per row, as TMEM hands them out,
// every store of a warp would touch 32 rows.
__device__ __forceinline__ void store_block(const GemmArgs& g, float* buf, const float* v, int64_t m0, int64_t n0,
                                            float scale, int sp, int lane) {
#pragma unroll
  for (int i = 0; i < 32; i++) buf[lane * kStagePitch + i] = v[i];
  __syncwarp();
  const int rows = (int)min((int64_t)32, g.M - m0);
  const int64_t n = n0 + lane;
  if (g.splits > 1) {
    float* d = g.partial + ((int64_t)sp * g.M + m0) * g.N + n;
    if (n < g.N)
      for (int r = 0; r < rows; r++) d[r * g.N] = buf[r * kStagePitch + lane];
  } else if (g.o.dtype != DT_F32 && !g.o.add && n0 + 32 <= g.N &&
             ((reinterpret_cast<uintptr_t>(g.o.c) | (uintptr_t)(g.o.ld * 2)) & 3u) == 0) {
    // 16-bit results in pairs, two rows at a time
    const int c = (lane & 15) * 2;
    for (int r = lane >> 4; r < rows; r += 2) {
      const float a = __fmul_rn(buf[r * kStagePitch + c], scale), b = __fmul_rn(buf[r * kStagePitch + c + 1], scale);
      const uint32_t w = g.o.dtype == DT_F16 ? f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16
                                             : f32_to_bf16_bits(a) | (uint32_t)f32_to_bf16_bits(b) << 16;
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(g.o.c) + (m0 + r) * g.o.ld + n0 + c) = w;
    }
  } else if (n < g.N) {
    for (int r = 0; r < rows; r++) finish(g.o, scale, m0 + r, n, buf[r * kStagePitch + lane]);
  }
  __syncwarp();
}

template <bool AMN, bool BMN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const GemmArgs g) {
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const uint32_t smem = (sptr(dyn) + 1023u) & ~1023u;
  const uint32_t full = sptr(bars), empty = full + 8 * kStages, tfull = empty + 8 * kStages, tempty = tfull + 16,
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
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sptr(&tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;
  const int units = g.tiles_m * g.tiles_n * g.splits;

  if (warp == 0 && lane == 0) {
    int it = 0;
    const uint32_t lead = in_cta(full, 0);
    bool ok = true;
    for (int u = pair; u < units && ok && !*abort; u += pairs) {
      int tm, tn;
      const int sp = u % g.splits;
      tile_at(g, u / g.splits, tm, tn);
      const int s1 = split_at(g, sp + 1);
      const int am = tm * kBM + rank * kHalf, bn = tn * kBN + rank * kHalf;
      for (int s = split_at(g, sp); s < s1; s++, it++) {
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
        const unsigned long long t0 = now_ns();
        while (!mbar_try(full + 8 * (i % kStages), (i / kStages) & 1) && now_ns() - t0 < kGemmWaitNs) {
        }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // D float32, A and B bfloat16, majors, N, M
    constexpr uint32_t idesc = 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)AMN << 15 | (uint32_t)BMN << 16 |
                               (uint32_t)(kBN >> 3) << 17 | (uint32_t)(kBM >> 4) << 24;
    int it = 0, chunk = 0;
    bool ok = true;
    for (int u = pair; u < units && ok && !*abort; u += pairs) {
      const int sp = u % g.splits, s1 = split_at(g, sp + 1);
      for (int c = split_at(g, sp); c < s1 && ok; c += kChunk64, chunk++) {
        const int buf = chunk & 1;
        if (chunk >= 2 && !(ok = mbar_wait(tempty + 8 * buf, (chunk / 2 - 1) & 1, abort))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int ce = min(c + kChunk64, s1);
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
      const unsigned long long t0 = now_ns();
      while (!mbar_try(drain, 0) && now_ns() - t0 < kGemmWaitNs) {
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + half * (kBN / 2);
    const uint32_t done = in_cta(tempty, 0);
    float* buf32 = reinterpret_cast<float*>(dyn + (smem - sptr(dyn)) + kStages * kStageBytes) + (warp - 4) * 32 * kStagePitch;
    const float scale = out_scale(g.o);
    int chunk = 0;
    bool ok = true;
    for (int u = pair; u < units && ok && !*abort; u += pairs) {
      int tm, tn;
      const int sp = u % g.splits, s1 = split_at(g, sp + 1);
      tile_at(g, u / g.splits, tm, tn);
      float acc[kBN / 2];
#pragma unroll
      for (int i = 0; i < kBN / 2; i++) acc[i] = 0.0f;
      for (int c = split_at(g, sp); c < s1; c += kChunk64, chunk++) {
        const int buf = chunk & 1;
        if (!(ok = mbar_wait(tfull + 8 * buf, (chunk / 2) & 1, abort))) break;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int j = 0; j < kBN / 2; j += 16) {
          uint32_t v[16];
          asm volatile(
              "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
              : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
              : "r"(taddr + buf * kBN + j));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int i = 0; i < 16; i++) acc[j + i] = __fadd_rn(acc[j + i], __uint_as_float(v[i]));
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(done + 8 * buf);
      }
      if (!ok) break;
      const int64_t m0 = (int64_t)tm * kBM + rank * kHalf + quarter * 32, n0 = (int64_t)tn * kBN + half * (kBN / 2);
#pragma unroll
      for (int i = 0; i < kBN / 2; i += 32)
        if (m0 < g.M && n0 + i < g.N) store_block(g, buf32, acc + i, m0, n0 + i, scale, sp, lane);
    }
  }
  __syncthreads();
  if (*abort && warp == 0) {  // what the other CTA's copies still do ends in this time
    const unsigned long long t0 = now_ns();
    while (now_ns() - t0 < 1000000ull) {
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// the splits' sums, added in their order; four columns per thread
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* __restrict__ partial, int splits, int64_t M, int64_t N,
                                                        LinearOut o) {
  const float scale = out_scale(o);
  const int64_t mn = M * N;
  for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
    const int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= N) continue;
    const float* s = partial + m * N + n;
    float v[4];
    const int w = (int)min((int64_t)4, N - n);
    if ((N & 3) == 0) {
      float4 t = __ldcs(reinterpret_cast<const float4*>(s));
      v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
      for (int i = 1; i < splits; i++) {
        t = __ldcs(reinterpret_cast<const float4*>(s + i * mn));
        v[0] = __fadd_rn(v[0], t.x), v[1] = __fadd_rn(v[1], t.y);
        v[2] = __fadd_rn(v[2], t.z), v[3] = __fadd_rn(v[3], t.w);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = k < w ? s[k] : 0.0f;
      for (int i = 1; i < splits; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (k < w) v[k] = __fadd_rn(v[k], s[i * mn + k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < w) finish(o, scale, m, n + k, v[k]);
  }
}

// A wait for a barrier that nothing arrives at (the time-out path's test).
__global__ void wait_selftest_kernel(unsigned long long limit) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  abort_flag = 0;
  mbar_init(sptr(&bar), 1);
  mbar_wait(sptr(&bar), 0, &abort_flag, limit);
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
  int planes, steps, tiles_m, tiles_n, splits;
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
  // fewer tiles than pairs of SMs: the reduction is split so that every pair
  // has a part, of one chunk at least
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, total = (int64_t)p.steps * p.planes;
  p.splits = 1;
  if (tiles < sms / 2) {
    const int64_t most = (total + kChunk64 - 1) / kChunk64;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(sms / 2 / tiles, most));
  }
  p.q_off = 0;
  p.a_off = up(p.q_off + p.qrows * p.qp * 2, 256);
  p.p_off = up(p.a_off + p.planes * p.arows * p.ap * 2, 256);
  p.bytes = p.p_off + (p.splits > 1 ? up((int64_t)p.splits * p.M * p.N * 4, 256) : 0);
  return p;
}

int grid_for(int64_t threads, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, (int64_t)sms * 8));
}

template <int KIND>
cudaError_t unpack_w4(const LinearArgs& a, const Plan& p, uint16_t* out, int sms, cudaStream_t st) {
  if (a.in % W4<KIND>::BE == 0) {
    const int64_t n = a.out * a.in;
    unpack_w4_flat_kernel<KIND><<<grid_for(n / 8, sms), 256, 0, st>>>(a.q, n, out);
  } else {
    unpack_w4_rows_kernel<KIND><<<grid_for(p.qrows * p.qp / 8, sms), 256, 0, st>>>(a.q, p.qrows, p.qcols, p.qp, out);
  }
  return cudaGetLastError();
}

template <bool AMN, bool BMN>
cudaError_t run_gemm(const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& g, int sms, cudaStream_t st) {
  static bool set[64] = {false};  // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(gemm_kernel<AMN, BMN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  const int64_t units = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  gemm_kernel<AMN, BMN><<<(unsigned)std::min<int64_t>(units, sms / 2) * 2, kGemmThreads, kGemmSmem, st>>>(ma, mb, g);
  return cudaGetLastError();
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

cudaError_t launch_wait_selftest(unsigned long long limit_ns, cudaStream_t st) {
  wait_selftest_kernel<<<1, 1, 0, st>>>(limit_ns);
  return cudaGetLastError();
}

int64_t gemm_workspace(const LinearArgs& a, int sms) { return make_plan(a, sms).bytes; }

cudaError_t launch_gemm(const LinearArgs& a, void* ws, int sms, cudaStream_t st) {
  const Plan p = make_plan(a, sms);
  uint8_t* base = static_cast<uint8_t*>(ws);
  uint16_t* q16 = reinterpret_cast<uint16_t*>(base + p.q_off);
  cudaError_t e;
  if (a.op == LIN_WGRAD) {
    const int64_t n16 = p.qrows * p.qp / 16;
    if (a.kind == A8_E4M3)
      unpack_a8_kernel<A8_E4M3><<<grid_for(n16, sms), 256, 0, st>>>(a.q, a.scales, n16, q16);
    else
      unpack_a8_kernel<A8_E5M2><<<grid_for(n16, sms), 256, 0, st>>>(a.q, a.scales, n16, q16);
    e = cudaGetLastError();
  } else if (a.kind == Q_MXFP4) {
    e = unpack_w4<Q_MXFP4>(a, p, q16, sms, st);
  } else if (a.kind == Q_MXFP4_OCP) {
    e = unpack_w4<Q_MXFP4_OCP>(a, p, q16, sms, st);
  } else {  // the tensor scale of ODY_Q_NVFP4_TENSOR is applied to the sums
    e = unpack_w4<Q_NVFP4>(a, p, q16, sms, st);
  }
  if (e != cudaSuccess) return e;
  // bfloat16 rows that TMA can read are used where they lie
  const void* abase = a.a;
  int64_t apitch = a.lda, aplane = up(p.arows * a.lda, 8);
  if (a.a_dtype != DT_BF16 || (reinterpret_cast<uintptr_t>(a.a) & 15u) || a.lda % 8) {
    uint16_t* a16 = reinterpret_cast<uint16_t*>(base + p.a_off);
    const int64_t es = a.a_dtype == DT_F32 ? 4 : 2;
    const int wide = (reinterpret_cast<uintptr_t>(a.a) & 15u) == 0 && (a.lda * es) % 16 == 0;
    apitch = p.ap, aplane = p.arows * p.ap;
    const int grid = grid_for(p.arows * p.ap / 8, sms);
    if (a.a_dtype == DT_F32)
      pack_planes_kernel<DT_F32><<<grid, 256, 0, st>>>(a.a, p.arows, p.acols, a.lda, apitch, aplane, a16, wide);
    else if (a.a_dtype == DT_F16)
      pack_planes_kernel<DT_F16><<<grid, 256, 0, st>>>(a.a, p.arows, p.acols, a.lda, apitch, aplane, a16, wide);
    else
      pack_planes_kernel<DT_BF16><<<grid, 256, 0, st>>>(a.a, p.arows, p.acols, a.lda, apitch, aplane, a16, wide);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    abase = a16;
  }
  const bool amn = a.op == LIN_WGRAD, bmn = a.op != LIN_FORWARD;
  CUtensorMap ma, mb;
  if ((e = make_map(&ma, abase, p.acols, p.arows, p.planes, apitch, aplane, amn ? kBK : kHalf)) != cudaSuccess) return e;
  if ((e = make_map(&mb, q16, p.qcols, p.qrows, 1, p.qp, p.qrows * p.qp, bmn ? kBK : kHalf)) != cudaSuccess) return e;
  GemmArgs g;
  g.o = a.o;
  g.M = p.M, g.N = p.N;
  g.tiles_m = p.tiles_m, g.tiles_n = p.tiles_n;
  g.steps = p.steps, g.planes = p.planes, g.splits = p.splits;
  g.partial = reinterpret_cast<float*>(base + p.p_off);
  if (a.op == LIN_FORWARD)
    e = run_gemm<false, false>(ma, mb, g, sms, st);
  else if (a.op == LIN_DGRAD)
    e = run_gemm<false, true>(ma, mb, g, sms, st);
  else
    e = run_gemm<true, true>(ma, mb, g, sms, st);
  if (e != cudaSuccess || p.splits == 1) return e;
  const int64_t jx = (p.N + 1023) / 1024;
  gemm_join_kernel<<<dim3((unsigned)jx, (unsigned)std::min<int64_t>(p.M, 65535)), 256, 0, st>>>(g.partial, p.splits, p.M,
                                                                                               p.N, a.o);
  return cudaGetLastError();
}

}  // namespace ody
