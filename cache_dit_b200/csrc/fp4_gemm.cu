// 4-bit microscaled product for sm_100a: out[m, n] = act(sum_k A[m, k] W[n, k] + bias[n])  (formats: fp4.cuh)
//
// The tensor core multiplies the e2m1 codes and applies both operands' block scales itself (tcgen05.mma with
// .block_scale, K = 64 per instruction), so the sum over all blocks stays one fp32 accumulation in tensor memory; the
// row scales of nvfp4, the bias and the optional tanh-GELU are applied in the epilogue.
//
//   * operands and their block scales by TMA into a ring of shared-memory stages of 256 columns (128 bytes) of K;
//     block scales go on to tensor memory (tcgen05.cp, 32 rows x 16 bytes broadcast to the four lane quarters);
//   * CG = 2: a pair of SMs works on a 256 x bn tile (each CTA loads 128 rows of A, half of the weight tile, and the
//     weight tile's scales whole, since each tensor core needs them); CG = 1: one SM, 128 x bn;
//   * two accumulators in tensor memory, so that a tile's epilogue overlaps the next tile's main loop.  Two of 256
//     columns leave no room for the scales (512 columns in all): at bn = 256 the second starts at column 160 and the
//     two share 96 columns.  The epilogue reads those 96 columns into registers first and hands them over; all that
//     the next tile's MMAs wait for is that read.
//   * one row: no tile; the weights are streamed once by the CUDA cores (fp4_gemv_kernel).
//
// Warp roles (352 threads): warp 0 = TMA producer, warp 1 = tensor memory owner and MMA issuer, warps 2..9 = epilogue (two
// per 32 rows, half of the columns each: the last tile's epilogue has nothing to hide under), warp 10 = block scales to
// tensor memory.
// Every wait is bounded (bounded_wait): on expiry the roles drain, tensor memory is freed and the kernel returns.
#include <cuda_fp16.h>

#include <atomic>
#include <cstdlib>

#include "fp4.cuh"
#include "tcgen05.cuh"

namespace cdb {

constexpr int F4_THREADS = 352;
constexpr int F4_EPI_WARP0 = 2;
constexpr int F4_EPI_THREADS = 256;
constexpr int F4_SCALE_WARP = 10;
constexpr int F4_MAX_STAGES = 8;
constexpr int F4_MAX_SLOTS = 8;
constexpr int F4_MAX_BN = 256;
constexpr int F4_A_BYTES = 128 * 128;     // 128 rows of one step's codes
constexpr uint32_t F4_TMEM_COLS = 512;
constexpr uint32_t F4_SHARED_COL = 160;   // where the second accumulator starts when bn = 256
constexpr int F4_BLOCK_BYTES = 32 * 64 * 2;                      // one staged block of output: 32 rows x 64 columns
constexpr int F4_STAGING_BYTES = (F4_EPI_THREADS / 32) * F4_BLOCK_BYTES;
constexpr int F4_SMEM_LIMIT = 232448;

struct __align__(8) F4Barriers {
  uint64_t full[F4_MAX_STAGES];
  uint64_t empty[F4_MAX_STAGES];
  uint64_t sf_full[F4_MAX_SLOTS];  // block scales of a step are in tensor memory
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  volatile int abort_flag;
};
constexpr int F4_FIXED_BYTES = 1024 + F4_STAGING_BYTES + F4_MAX_BN * 8 + (int)sizeof(F4Barriers);

struct F4Params {
  CUtensorMap map_a, map_w, map_sa, map_sw, map_out;
  const float* ra;  // row scales, or null (mxfp4)
  const float* rw;
  const void* bias;
  int M, N;
  int m_tiles, n_tiles, k_steps, group_m, num_tiles;
  int stages, stage_bytes, gelu;
  uint32_t sf_col;
  int slots;
  uint32_t idesc;
};

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* map, uint32_t bar_cluster_addr, void* dst, int c0,
                                                 int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(bar_cluster_addr), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// tcgen05 instructions of a whole, converged warp: each elects its issuing lane itself.  Under a branch on an elected
// lane every operand had to be made uniform by hand of the compiler, about 60 clocks an instruction.
#define CDB_ELECTED(text) "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\t" text "\n\t}"
// 32 rows x 16 bytes of shared memory -> 4 tensor memory columns, the same in all four lane quarters (CG = 2: in both
// CTAs, each from its own shared memory).
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (CG == 2) asm volatile(CDB_ELECTED("@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;") ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile(CDB_ELECTED("@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;") ::"r"(tmem), "l"(desc) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit_warp(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(CDB_ELECTED("@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;")
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile(CDB_ELECTED("@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];") ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit_own(uint32_t bar) {  // to this CTA's barrier alone
  if constexpr (CG == 2)
    asm volatile(CDB_ELECTED("@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];") ::"r"(bar) : "memory");
  else
    asm volatile(CDB_ELECTED("@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];") ::"r"(bar) : "memory");
}
#define CDB_F4_MMA(CG_, KIND_)                                                                                      \
  asm volatile(CDB_ELECTED("setp.ne.b32 p, %6, 0;\n\t"                                                              \
                           "@e tcgen05.mma.cta_group::" CG_ ".kind::" KIND_ " [%0], %1, %2, %3, [%4], [%5], p;")     \
               ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                \
               : "memory")
template <int CG, bool NV>
__device__ __forceinline__ void mma_f4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 1 && NV) CDB_F4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  if constexpr (CG == 1 && !NV) CDB_F4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  if constexpr (CG == 2 && NV) CDB_F4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
  if constexpr (CG == 2 && !NV) CDB_F4_MMA("2", "mxf4.block_scale.scale_vec::2X");
}
// Block-scaled instruction descriptor: [4,6) scale id of B, [7,10) A = e2m1 (1), [10,13) B = e2m1 (1), [17,23) N >> 3,
// bit 23 scale type (0 = e4m3, 1 = e8m0), [24,29) M >> 4, [29,31) scale id of A.  The scale id picks the half of a
// tensor memory word that holds an instruction's two e8m0 scales (0 or 2).
constexpr uint32_t f4_idesc(int m, int n, bool nv) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((nv ? 0u : 1u) << 23) | ((uint32_t)(m >> 4) << 24);
}
// Descriptor of one 512-byte scale tile: no swizzle, groups of 8 rows x 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t scale_tile_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// Position in the ring of stages: index and phase bit, advanced without the divisions that would sit in every step's
// serial chain (they took more clocks than a step's MMAs).
struct RingPos {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
};
// M fastest inside groups of `group_m` row tiles, so a wave shares weight tiles and a bounded set of A panels in L2.
__device__ __forceinline__ void f4_tile_coords(int tile, const F4Params& p, int& mi, int& ni) {
  const int per_group = p.group_m * p.n_tiles;
  const int group = tile / per_group;
  const int first_m = group * p.group_m;
  const int rows = min(p.group_m, p.m_tiles - first_m);
  const int in_group = tile - group * per_group;
  mi = first_m + in_group % rows;
  ni = in_group / rows;
}
__device__ __forceinline__ bool f4_epi_all(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)pred), "n"(F4_EPI_THREADS)
      : "memory");
  return r != 0;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (__is_same(T, __nv_bfloat16)) {
    return pack_bf16x2(lo, hi);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// The scale of an activation row in two factors, low <= 1 <= high (a NaN is in high).  An accumulator is in units of both
// operands' scaled codes, up to 2^37: times a large row scale it may be beyond fp32 where the weight row's small scale would
// bring it back, and the other way round with small ones.  low, then the weight's scale, then high: no step is larger than
// the result, and none but the last smaller than 2^-120.
struct RowScale {
  float low, high;
  __device__ __forceinline__ explicit RowScale(float s) : low(s < 1.f ? s : 1.f), high(s < 1.f ? 1.f : s) {}
};

// One staged block: 32 rows x 64 columns starting at local column `c0` of the tile, from 2 x 32 accumulator registers.
template <typename T>
__device__ __forceinline__ void f4_store_block(const F4Params& p, uint8_t* block,
                                               const uint32_t (&lo)[32], const uint32_t (&hi)[32], int c0, int n0,
                                               int row0, const RowScale& rs, const float2* s_col, int lane) {
  if (n0 + c0 >= p.N) return;
  if (lane == 0) bulk_wait_group_read<0>();  // the store before this one is done reading
  __syncwarp();
  uint8_t* rowp = block + lane * 128;
#pragma unroll
  for (int g = 0; g < 8; ++g) {  // 8 columns = one 16-byte chunk
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = g * 8 + 2 * j;
      const float4 sb = *reinterpret_cast<const float4*>(s_col + c0 + c);  // (scale, bias) of two columns
      const float a0 = __uint_as_float(c < 32 ? lo[c & 31] : hi[c & 31]);
      const float a1 = __uint_as_float(c < 32 ? lo[(c + 1) & 31] : hi[(c + 1) & 31]);
      float v0 = fmaf(a0 * rs.low * sb.x, rs.high, sb.y), v1 = fmaf(a1 * rs.low * sb.z, rs.high, sb.w);
      if (p.gelu) {
        v0 = gelu_tanh(v0);
        v1 = gelu_tanh(v1);
      }
      w[j] = pack2<T>(v0, v1);
    }
    *reinterpret_cast<uint4*>(rowp + ((g ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(&p.map_out, block, n0 + c0, row0);
    bulk_commit_group();
  }
  __syncwarp();  // what follows may be the whole warp's (a load from tensor memory, a barrier)
}

template <int CG, int BN, bool NV, typename T>
__global__ void __launch_bounds__(F4_THREADS, 1) fp4_gemm_kernel(const __grid_constant__ F4Params p, int32_t* status_word) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_staging = smem + p.stages * p.stage_bytes;  // a multiple of 1024
  float2* s_col = reinterpret_cast<float2*>(s_staging + F4_STAGING_BYTES);
  F4Barriers* gb = reinterpret_cast<F4Barriers*>(s_col + F4_MAX_BN);

  constexpr int TILES = NV ? 4 : 2;  // scale tiles of one step and panel
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform to the compiler as well
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;  // 0 owns the shared barriers and issues the MMAs
  const int first = CG == 2 ? blockIdx.x >> 1 : blockIdx.x;
  const int step = CG == 2 ? gridDim.x >> 1 : gridDim.x;
  constexpr int bn = BN;
  constexpr int PANELS = BN > 128 ? BN / 128 : 1;  // of 128 weight rows: one tile's scales
  constexpr uint32_t sfa_off = F4_A_BYTES + BN / CG * 128;
  constexpr uint32_t sfb_off = sfa_off + TILES * 512;
  constexpr uint32_t SLOT_COLS = TILES * 4 * (1 + PANELS);
  constexpr bool shared_acc = BN == F4_MAX_BN;
  constexpr uint32_t acc1 = shared_acc ? F4_SHARED_COL : BN;
  const int stages = p.stages;
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    for (int s = 0; s < F4_MAX_STAGES; ++s) {
      mbar_init(&gb->full[s], 1);
      mbar_init(&gb->empty[s], 1);
    }
    for (int i = 0; i < F4_MAX_SLOTS; ++i) mbar_init(&gb->sf_full[i], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&gb->acc_full[b], 1);
      mbar_init(&gb->acc_empty[b], CG * (F4_EPI_THREADS / 32));
    }
    gb->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&gb->tmem_base)), "r"(F4_TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&gb->tmem_base)), "r"(F4_TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();  // the peer's barriers exist before anything is signalled across the pair
  tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, gb->tmem_base, 0);
  pdl_wait_prior();  // what is before this ran beside the end of the kernel that wrote the operands

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      RingPos at;
      uint32_t issued = 0;
      bool ok = true;
      constexpr uint32_t tx = CG * (sfb_off + PANELS * TILES * 512);  // both CTAs' bytes of one stage
      for (int tile = first; tile < p.num_tiles && ok; tile += step) {
        int mi, ni;
        f4_tile_coords(tile, p, mi, ni);
        const int m0 = mi * (128 * CG) + (int)rank * 128;
        const int n0 = ni * bn;
        const int w0 = n0 + (CG == 2 ? (int)rank * (bn >> 1) : 0);
        for (int kb = 0; kb < p.k_steps; ++kb, at.next(stages), ++issued) {
          const int s = at.stage;
          ok = bounded_wait(&gb->empty[s], at.phase ^ 1u, &gb->abort_flag, status_word, 21);
          if (!ok) break;
          uint8_t* dst = smem + s * p.stage_bytes;
          if constexpr (CG == 2) {
            if (rank == 0) mbar_expect_tx(&gb->full[s], tx);
            const uint32_t full = map_to_cta(smem_u32(&gb->full[s]), 0);
            tma_load_2d_pair(&p.map_a, full, dst, kb * 128, m0);
            tma_load_2d_pair(&p.map_w, full, dst + F4_A_BYTES, kb * 128, w0);
            tma_load_3d_pair(&p.map_sa, full, dst + sfa_off, 0, kb * TILES * 4, m0 >> 7);
            tma_load_3d_pair(&p.map_sw, full, dst + sfb_off, 0, kb * TILES * 4, n0 >> 7);
          } else {
            mbar_expect_tx(&gb->full[s], tx);
            tma_load_2d(&p.map_a, &gb->full[s], dst, kb * 128, m0);
            tma_load_2d(&p.map_w, &gb->full[s], dst + F4_A_BYTES, kb * 128, w0);
            tma_load_3d(&p.map_sa, &gb->full[s], dst + sfa_off, 0, kb * TILES * 4, m0 >> 7);
            tma_load_3d(&p.map_sw, &gb->full[s], dst + sfb_off, 0, kb * TILES * 4, n0 >> 7);
          }
        }
      }
      // A CTA may not retire while copies into its shared memory are in flight or while MMAs read it: wait (bounded,
      // also after an abort) until the MMAs released every stage used.
      const uint64_t t0 = global_timer_ns();
      for (uint32_t j = (issued > (uint32_t)stages ? issued - stages : 0); j < issued; ++j) {
        while (!mbar_try_wait(&gb->empty[j % stages], (j / stages) & 1u)) {
          if (global_timer_ns() - t0 > BARRIER_LIMIT_NS) break;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (rank == 0) {  // the whole warp waits, one elected lane issues
      const uint32_t smem_base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      RingPos at, slot;
      uint32_t n_tile = 0;
      bool ok = true;
      for (int tile = first; tile < p.num_tiles && ok; tile += step, ++n_tile) {
        const uint32_t buf = n_tile & 1u;
        // Separate accumulators: tile n_tile - 2 has left this one.  Shared columns: tile n_tile - 1 has left them
        // (and n_tile - 2 everything, since the epilogue takes tiles in order).
        if (!shared_acc) {
          ok = __all_sync(0xffffffffu, bounded_wait(&gb->acc_empty[buf], ((n_tile >> 1) & 1u) ^ 1u, &gb->abort_flag, status_word, 22));
        } else if (n_tile > 0) {
          ok = __all_sync(0xffffffffu, bounded_wait(&gb->acc_empty[buf ^ 1u], ((n_tile - 1) >> 1) & 1u, &gb->abort_flag, status_word, 22));
        }
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t tmem_d = tmem_base + buf * acc1;
        int mi, ni;
        f4_tile_coords(tile, p, mi, ni);
        // a 64-column tile may be the second half of its panel of 128 weight rows: scales two columns on
        const uint32_t sfb_skip = (uint32_t)((ni * bn) & 127) >> 5;
        for (int kb = 0; kb < p.k_steps; ++kb, at.next(stages)) {
          const int s = at.stage;
          ok = __all_sync(0xffffffffu, bounded_wait(&gb->full[s], at.phase, &gb->abort_flag, status_word, 23));
          if (!ok) break;
          ok = __all_sync(0xffffffffu, bounded_wait(&gb->sf_full[slot.stage], slot.phase, &gb->abort_flag, status_word, 24));
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t base = smem_base + (uint32_t)s * (uint32_t)p.stage_bytes;
          const uint32_t sfa = tmem_base + p.sf_col + (uint32_t)slot.stage * SLOT_COLS;
          const uint32_t sfb = sfa + TILES * 4;
          const uint64_t adesc = make_kmajor_sw128_desc(base);
          const uint64_t bdesc = make_kmajor_sw128_desc(base + F4_A_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // 64 columns = 32 bytes: +2 in the (address >> 4) field
            const int j = NV ? k : k >> 1;
            const uint32_t id = NV ? 0u : (uint32_t)(k & 1) * 2u;
            mma_f4<CG, NV>(tmem_d, adesc + 2 * k, bdesc + 2 * k, p.idesc | (id << 4) | (id << 29), sfa + j * 4,
                           sfb + j * PANELS * 4 + sfb_skip, (kb | k) != 0 ? 1u : 0u);
          }
          commit_warp<CG>(smem_u32(&gb->empty[s]));
          slot.next(p.slots);
        }
        if (ok) commit_warp<CG>(smem_u32(&gb->acc_full[buf]));
      }
    }
    __syncwarp();
  } else if (warp == F4_SCALE_WARP) {
    // ---------------- block scales: shared memory -> tensor memory, ahead of the MMAs ----------------
    // A warp of its own: in the MMA issuer these copies and the wait for their slot sat between two steps' MMAs.
    if (rank == 0) {
      const uint32_t smem_base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      RingPos at, old, slot;  // `old`: the step whose scale slot is written next
      bool ok = true, slots_used = false;
      for (int tile = first; tile < p.num_tiles && ok; tile += step) {
        for (int kb = 0; kb < p.k_steps; ++kb, at.next(stages)) {
          // The slot's last readers are the MMAs of `slots` steps ago: they have retired when their stage is released.
          if (slots_used) {
            ok = __all_sync(0xffffffffu, bounded_wait(&gb->empty[old.stage], old.phase, &gb->abort_flag, status_word, 26));
            if (!ok) break;
            old.next(stages);
          }
          ok = __all_sync(0xffffffffu, bounded_wait(&gb->full[at.stage], at.phase, &gb->abort_flag, status_word, 27));
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t base = smem_base + (uint32_t)at.stage * (uint32_t)p.stage_bytes;
          const uint32_t sfa = tmem_base + p.sf_col + (uint32_t)slot.stage * SLOT_COLS;
          const uint32_t sfb = sfa + TILES * 4;
#pragma unroll
          for (int j = 0; j < TILES; ++j) {
            copy_scales<CG>(sfa + j * 4, scale_tile_desc(base + sfa_off + j * 512));
#pragma unroll
            for (int q = 0; q < PANELS; ++q)
              copy_scales<CG>(sfb + (j * PANELS + q) * 4, scale_tile_desc(base + sfb_off + (q * TILES + j) * 512));
          }
          commit_own<CG>(smem_u32(&gb->sf_full[slot.stage]));
          slot.next(p.slots);
          slots_used = slots_used || slot.stage == 0;
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue: this CTA's 128 rows x bn columns ----------------
    const int quarter = warp & 3;
    const int et = threadIdx.x - F4_EPI_WARP0 * 32;
    const int half = (warp - F4_EPI_WARP0) >> 2;  // of the tile's columns
    uint8_t* staging = s_staging + (warp - F4_EPI_WARP0) * F4_BLOCK_BYTES;
    const T* bias = static_cast<const T*>(p.bias);
    uint32_t n_tile = 0;
    bool ok = true;
    for (int tile = first; tile < p.num_tiles && ok; tile += step, ++n_tile) {
      int mi, ni;
      f4_tile_coords(tile, p, mi, ni);
      const int row0 = mi * (128 * CG) + (int)rank * 128 + quarter * 32;
      const int n0 = ni * bn;
      const uint32_t buf = n_tile & 1u;
      asm volatile("bar.sync 1, %0;" ::"n"(F4_EPI_THREADS) : "memory");  // the last tile's readers of s_col are done
      for (int c = et; c < bn; c += F4_EPI_THREADS) {
        const int col = n0 + c;
        float2 v = make_float2(0.f, 0.f);
        if (col < p.N) {
          v.x = p.rw != nullptr ? __ldg(p.rw + col) : 1.f;
          if (bias != nullptr) v.y = (float)bias[col];
        }
        s_col[c] = v;
      }
      ok = bounded_wait(&gb->acc_full[buf], (n_tile >> 1) & 1u, &gb->abort_flag, status_word, 25);
      __syncwarp();
      ok = f4_epi_all(ok);  // publishes s_col, and makes the decision to go on the same in all its warps
      if (!ok) break;
      tcgen05_fence_after();
      const int row = row0 + lane;
      const RowScale rs(row < p.M && p.ra != nullptr ? __ldg(p.ra + row) : 1.f);
      __syncwarp();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * acc1;
      const bool live = row0 < p.M;  // warp-uniform: some of the 32 rows exist
      auto release = [&] {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) mbar_arrive_cluster(map_to_cta(smem_u32(&gb->acc_empty[buf]), 0));
          else mbar_arrive(&gb->acc_empty[buf]);
        }
        __syncwarp();
      };
      auto plain_blocks = [&](int from, int to) {
#pragma unroll 1
        for (int c = from; c < to && n0 + c < p.N; c += 64) {
          uint32_t lo[32], hi[32];
          tmem_ld_32x32b_x32(taddr + c, lo);
          tmem_ld_32x32b_x32(taddr + c + 32, hi);
          tmem_ld_wait();
          f4_store_block<T>(p, staging, lo, hi, c, n0, row0, rs, s_col, lane);
        }
      };
      if constexpr (!shared_acc) {
        constexpr int split = bn > 64 ? bn / 2 : 64;
        if (live) plain_blocks(half ? split : 0, half ? bn : split);
        release();
      } else if (!live) {
        release();
      } else {
        // The columns that the other accumulator overlaps are 160..255 of the first and 0..95 of the second: all of them in
        // one half.
        if ((int)buf == half) {
          release();
          plain_blocks(half * 128, half * 128 + 128);
        } else {
          uint32_t s0[32], s1[32], s2[32], x[32];
          const uint32_t at = taddr + (buf == 0 ? F4_SHARED_COL : 0u);
          tmem_ld_32x32b_x32(at, s0);
          tmem_ld_32x32b_x32(at + 32, s1);
          tmem_ld_32x32b_x32(at + 64, s2);
          tmem_ld_wait();
          release();
          if (buf == 0) {
            f4_store_block<T>(p, staging, s1, s2, 192, n0, row0, rs, s_col, lane);
            tmem_ld_32x32b_x32(taddr + 128, x);
            tmem_ld_wait();
            f4_store_block<T>(p, staging, x, s0, 128, n0, row0, rs, s_col, lane);
          } else {
            f4_store_block<T>(p, staging, s0, s1, 0, n0, row0, rs, s_col, lane);
            tmem_ld_32x32b_x32(taddr + 96, x);
            tmem_ld_wait();
            f4_store_block<T>(p, staging, s2, x, 64, n0, row0, rs, s_col, lane);
          }
        }
        tcgen05_fence_before();  // orders these reads before the next barrier, behind which MMAs may overwrite them
      }
    }
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  tcgen05_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();  // neither CTA leaves while the other may still touch its memory
  if (warp == 1) {
    tcgen05_fence_after();
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(F4_TMEM_COLS) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(F4_TMEM_COLS) : "memory");
  }
}

// ---- one row ------------------------------------------------------------------------------------------------
// M = 1: a 128-row tile would be padding, and the weights (N * K * 9/16 bytes) are all there is to read.  A warp owns the
// four columns n, n + 32, n + 64, n + 96 whose block scales share 16 bytes; a lane takes 32 columns of K at a time: 16
// bytes of codes of each, one 16-byte load of scales, and the activations, from shared memory, once for all four.  The
// products of a block of 16 are multiples of 0.25 and at most 36: eight of them sum exactly in f16 (at most 288), so the two
// halves of a packed f16 accumulator hold the sum exactly; blocks are summed in fp32.
// Where the columns are too few to fill the SMs with warps, `split` warps of a block share their columns and take every
// split-th 32 chunks of K each; their sums are added in order.
// From two rows on the tile kernels are faster (4 x 30720 x 5120: 29 us against 50 us of this kernel with four rows).
constexpr int F4V_THREADS = 256;
__host__ __device__ constexpr size_t f4v_smem(int chunks) { return (size_t)chunks * (64 + 8); }  // f16 codes, two fp32 scales

// Scales of the two blocks of 16 of a chunk of 32 columns, from the word that holds its four (nvfp4: of 64 columns, mxfp4:
// of 128).
template <bool NV>
__device__ __forceinline__ float2 chunk_scales(uint32_t word, int c) {
  if constexpr (NV) {
    const uint32_t two = (c & 1) ? word >> 16 : word;
    return make_float2(e4m3_to_float(two & 0xffu), e4m3_to_float((two >> 8) & 0xffu));
  } else {
    const float s = e8m0_to_float((word >> ((c & 3) * 8)) & 0xffu);
    return make_float2(s, s);
  }
}

template <bool NV, typename T>
__global__ void __launch_bounds__(F4V_THREADS, 4)
    fp4_gemv_kernel(const uint8_t* __restrict__ a_codes, const uint8_t* __restrict__ a_scales, const float* __restrict__ ra,
                    const uint8_t* __restrict__ w_codes, const uint8_t* __restrict__ w_scales, const float* __restrict__ rw,
                    const T* __restrict__ bias, T* __restrict__ out, int N, int K, int split, int gelu) {
  pdl_launch_dependents();
  pdl_wait_prior();
  extern __shared__ __align__(16) uint8_t smem_raw[];
  constexpr int PER_WORD = NV ? 1 : 2;  // log2 of the chunks whose scales share a word
  const int chunks = K >> 5;            // of 32 columns = 16 bytes of codes
  const int64_t tiles = fp4_panel_tiles(K, NV);
  uint4* s_a = reinterpret_cast<uint4*>(smem_raw);             // [4][chunks]: 8 f16 codes each
  float2* s_s = reinterpret_cast<float2*>(s_a + 4 * chunks);   // [chunks]
  for (int c = threadIdx.x; c < chunks; c += F4V_THREADS) {
    const uint4 v = *(reinterpret_cast<const uint4*>(a_codes) + c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t f[4];
      e2m1x8_to_half2(w[j], f);
      s_a[j * chunks + c] = make_uint4(f[0], f[1], f[2], f[3]);
    }
    s_s[c] = chunk_scales<NV>(*reinterpret_cast<const uint32_t*>(a_scales + fp4_scale_word(0, c >> PER_WORD, tiles)), c);
    if constexpr (!NV) {  // one scale for the 32 columns, 2^-127 .. 2^127: in two factors, as a row scale
      const RowScale s(s_s[c].x);
      s_s[c] = make_float2(s.low, s.high);
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp & (split - 1);
  const int g = blockIdx.x * (F4V_THREADS / 32 / split) + warp / split;
  // g < groups for every warp: the groups, a multiple of 32, are a whole number of blocks.
  const int n0 = (g >> 5) * 128 + (g & 31);
  const uint4* wrow[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) wrow[j] = reinterpret_cast<const uint4*>(w_codes + (int64_t)min(n0 + 32 * j, N - 1) * (K >> 1));
  const uint8_t* srow = w_scales + fp4_scale_word(n0, 0, tiles);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int c = part * 32 + lane; c < chunks; c += 32 * split) {
    const uint4 sw = __ldg(reinterpret_cast<const uint4*>(srow + (c >> PER_WORD) * 512));
    uint4 wv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) wv[j] = __ldcs(wrow[j] + c);
    const float2 as = s_s[c];
    uint4 av[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) av[j] = s_a[j * chunks + c];
    const uint32_t sword[4] = {sw.x, sw.y, sw.z, sw.w};
    auto h2 = [](const uint32_t& u) { return *reinterpret_cast<const __half2*>(&u); };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 ws = chunk_scales<NV>(sword[j], c);
      const uint32_t word[4] = {wv[j].x, wv[j].y, wv[j].z, wv[j].w};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t f0[4], f1[4];
        e2m1x8_to_half2(word[2 * b], f0);
        e2m1x8_to_half2(word[2 * b + 1], f1);
        __half2 t = __hmul2(h2(f0[0]), h2(av[2 * b].x));
        t = __hfma2(h2(f0[1]), h2(av[2 * b].y), t);
        t = __hfma2(h2(f0[2]), h2(av[2 * b].z), t);
        t = __hfma2(h2(f0[3]), h2(av[2 * b].w), t);
        t = __hfma2(h2(f1[0]), h2(av[2 * b + 1].x), t);
        t = __hfma2(h2(f1[1]), h2(av[2 * b + 1].y), t);
        t = __hfma2(h2(f1[2]), h2(av[2 * b + 1].z), t);
        t = __hfma2(h2(f1[3]), h2(av[2 * b + 1].w), t);
        const float2 d = __half22float2(t);
        if constexpr (NV) acc[j] = fmaf(d.x + d.y, b ? ws.y * as.y : ws.x * as.x, acc[j]);
        else acc[j] = fmaf((d.x + d.y) * as.x * ws.x, as.y, acc[j]);  // the scales' product alone may be beyond fp32
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = warp_sum(acc[j]);
  if (split > 1) {
    __shared__ float4 s_part[F4V_THREADS / 32];
    if (lane == 0) s_part[warp] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (part != 0) return;
    for (int i = 1; i < split; ++i) {
      const float4 more = s_part[warp + i];
      acc[0] += more.x;
      acc[1] += more.y;
      acc[2] += more.z;
      acc[3] += more.w;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // lane j writes column j
    const int n = n0 + 32 * j;
    if (lane == j && n < N) {
      const float cs = rw != nullptr ? __ldg(rw + n) : 1.f;
      const RowScale rs(ra != nullptr ? __ldg(ra) : 1.f);
      float v = fmaf(acc[j] * rs.low * cs, rs.high, bias != nullptr ? (float)bias[n] : 0.f);
      if (gelu) v = gelu_tanh(v);
      out[n] = (T)v;
    }
  }
}

// ---- host side -----------------------------------------------------------------------------------------------
static bool f4_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, bool swizzle) {
  const EncodeTiledFn fn = tensor_map_encoder();
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn != nullptr &&
         fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static bool f4_code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols / 2, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols / 2};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  return f4_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, true);
}
// Scales as [panels, 4 * tiles, 128 bytes]; one step is a box of 4 * TILES lines of `panels` panels.
static bool f4_scale_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, bool nv, int panels) {
  const cuuint64_t lines = (cuuint64_t)fp4_panel_tiles(cols, nv) * 4;
  const cuuint64_t dims[3] = {128, lines, (cuuint64_t)(rows + 127) / 128}, strides[2] = {128, lines * 128};
  const cuuint32_t box[3] = {128, nv ? 16u : 8u, (cuuint32_t)panels};
  return f4_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box, false);
}

struct F4Plan {
  bool pair;
  int bn;
};
// Tuning / testing knob: 0 = chosen by size, else the tile's columns, negative for a CTA pair's.
static std::atomic<int> g_f4_tile{0};
// Tile shape of a launch, by a cost in steps of a 256-column pair tile (0.55 us): waves of tiles x steps x what a step
// of that shape costs, plus what a launch of it costs whatever K (filling the ring, the last tile's epilogue).  Fitted
// to nvfp4 launches with cold weights (M, N, K: 4608 x 5120 x 13824, 1153 x 12288 x 5120, 512 x 13824 x 5120, 77 x 5120
// x 4096): pair 256 / pair 128 / single 128 / single 64 take 141 / 213 / 211 / 417, 49 / 61 / 59 / 104,
// 27.7 / 29.4 / 28.6 / 51 and 13.8 / 11.0 / 10.2 / 10.0 us.
// Held against every shape on 18 launches of 2 to 16384 rows in both formats: within 2 % of the fastest, but for
// 4 x 30720 x 5120 (single 128 instead of pair 256: 4 % nvfp4, 9 % mxfp4) and 2000 x 5120 x 1536 (pair 256 instead of
// single 128: 17 % and 11 %).
static F4Plan f4_plan(int64_t M, int64_t N, int64_t K, int sms) {
  const struct { bool pair; int bn; double step, launch; } shapes[] = {
      {true, 256, 1.0, 9.0}, {true, 128, 0.82, 6.0}, {false, 128, 0.81, 5.5}, {false, 64, 0.72, 6.0}};
  const int64_t k_steps = (K + FP4_STEP_COLS - 1) / FP4_STEP_COLS;
  const int forced = g_f4_tile.load(std::memory_order_relaxed);
  if (forced != 0) return F4Plan{forced < 0, forced < 0 ? -forced : forced};
  F4Plan best{true, 256};
  double best_cost = 1e300;
  for (const auto& s : shapes) {
    if (s.pair && M <= 128) continue;
    const int64_t bm = s.pair ? 256 : 128;
    const int64_t tiles = ((M + bm - 1) / bm) * ((N + s.bn - 1) / s.bn);
    const int64_t slots = s.pair ? sms / 2 : sms;
    const double cost = (double)((tiles + slots - 1) / slots * k_steps) * s.step + s.launch;
    if (cost < best_cost) {
      best_cost = cost;
      best = F4Plan{s.pair, s.bn};
    }
  }
  return best;
}

template <int CG, int BN, bool NV, typename T>
static int f4_launch(F4Params& p, int32_t* status_word, cudaStream_t st) {
  static PerDevice attr_state;
  const cudaError_t attr_err = (cudaError_t)attr_state.get([]() -> int64_t {
    return (int64_t)cudaFuncSetAttribute(fp4_gemm_kernel<CG, BN, NV, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, F4_SMEM_LIMIT);
  });
  CDB_CUDA_CHECK(attr_err);
  const int slots = CG == 2 ? sm_count() / 2 : sm_count();
  const unsigned grid = (unsigned)((p.num_tiles < slots ? p.num_tiles : slots) * CG);
  CDB_CUDA_CHECK(launch_pdl_cluster(fp4_gemm_kernel<CG, BN, NV, T>, dim3(grid), dim3(F4_THREADS),
                                    (size_t)(F4_FIXED_BYTES + p.stages * p.stage_bytes), st, (unsigned)CG, p, status_word));
  return CDB_OK;
}

struct F4Matrix {  // mirrors `cdb_fp4_matrix` of the public header
  const void* codes;
  const void* block_scales;
  const float* row_scale;
};

template <bool NV, typename T>
static int f4_gemv(const F4Matrix& a, const F4Matrix& w, const void* bias, void* out, int64_t N, int64_t K, int gelu,
                   cudaStream_t st) {
  const size_t smem = f4v_smem((int)(K / 32));  // at most 36 KB: no opt-in
  // Four blocks an SM are resident: split K until there are as many, down to one load per lane.
  const int64_t warps = (N + 127) / 128 * 32;
  int split = 1;
  while (split < F4V_THREADS / 32 && warps * split < (int64_t)sm_count() * 4 * (F4V_THREADS / 32) && split * 64 <= K / 32) split *= 2;
  const int64_t want = warps * split / (F4V_THREADS / 32);  // warps is a multiple of 32: no rest
  CDB_CUDA_CHECK(launch_pdl(fp4_gemv_kernel<NV, T>, dim3((unsigned)want), dim3(F4V_THREADS), smem, st,
                            static_cast<const uint8_t*>(a.codes), static_cast<const uint8_t*>(a.block_scales), a.row_scale,
                            static_cast<const uint8_t*>(w.codes), static_cast<const uint8_t*>(w.block_scales), w.row_scale,
                            static_cast<const T*>(bias), static_cast<T*>(out), (int)N, (int)K, split, gelu));
  return CDB_OK;
}

template <bool NV, typename T>
static int f4_gemm(const F4Matrix& a, const F4Matrix& w, const void* bias, void* out, int64_t M, int64_t N, int64_t K,
                   int64_t ld_out, int gelu, int32_t* status_word, cudaStream_t st) {
  if (g_f4_tile.load(std::memory_order_relaxed) == 0 && M == 1) return f4_gemv<NV, T>(a, w, bias, out, N, K, gelu, st);
  const F4Plan plan = f4_plan(M, N, K, sm_count());
  const int cg = plan.pair ? 2 : 1, bn = plan.bn;
  const int panels = bn > 128 ? bn / 128 : 1;
  F4Params p{};
  const cuuint64_t odims[2] = {(cuuint64_t)N, (cuuint64_t)M}, ostrides[1] = {(cuuint64_t)ld_out * 2};
  const cuuint32_t obox[2] = {64, 32};
  if (!f4_code_map(&p.map_a, a.codes, M, K, 128) || !f4_code_map(&p.map_w, w.codes, N, K, bn / cg) ||
      !f4_scale_map(&p.map_sa, a.block_scales, M, K, NV, 1) || !f4_scale_map(&p.map_sw, w.block_scales, N, K, NV, panels) ||
      !f4_map(&p.map_out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, out, odims, ostrides, obox, true)) {
    set_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled");
    return CDB_ERR_CUDA;
  }
  p.ra = NV ? a.row_scale : nullptr;
  p.rw = NV ? w.row_scale : nullptr;
  p.bias = bias;
  p.M = (int)M;
  p.N = (int)N;
  p.m_tiles = (int)((M + 128 * cg - 1) / (128 * cg));
  p.n_tiles = (int)((N + bn - 1) / bn);
  p.k_steps = (int)((K + FP4_STEP_COLS - 1) / FP4_STEP_COLS);
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  if (tiles > INT32_MAX) return CDB_ERR_TOO_LARGE;
  p.num_tiles = (int)tiles;
  const int groups = (p.m_tiles + 15) / 16;
  p.group_m = p.m_tiles <= 24 ? p.m_tiles : (p.m_tiles + groups - 1) / groups;
  p.gelu = gelu != 0;
  p.idesc = f4_idesc(128 * cg, bn, NV);
  p.stage_bytes = F4_A_BYTES + bn / cg * 128 + (NV ? 4 : 2) * 512 * (1 + panels);
  const int fit = (F4_SMEM_LIMIT - F4_FIXED_BYTES) / p.stage_bytes;
  p.stages = fit < F4_MAX_STAGES ? fit : F4_MAX_STAGES;
  // Scale slots: what the accumulators leave of tensor memory, and no more than stages.  A slot's release is told by its stage's barrier, whose phase bit says nothing about a use more than one round of the ring ago.
  p.sf_col = bn == F4_MAX_BN ? F4_SHARED_COL + F4_MAX_BN : 2 * bn;
  const uint32_t fit_slots = (F4_TMEM_COLS - p.sf_col) / ((NV ? 16 : 8) * (1 + panels));
  p.slots = (int)fit_slots < p.stages ? (int)fit_slots : p.stages;
  if (plan.pair) return bn == 256 ? f4_launch<2, 256, NV, T>(p, status_word, st) : f4_launch<2, 128, NV, T>(p, status_word, st);
  return bn == 128 ? f4_launch<1, 128, NV, T>(p, status_word, st) : f4_launch<1, 64, NV, T>(p, status_word, st);
}

}  // namespace cdb

using namespace cdb;

extern "C" int cdb_tuning_set_fp4_tile(int pair, int cols) {
  if (cols != 0 && cols != 128 && cols != (pair ? 256 : 64)) return CDB_ERR_BAD_ARGUMENT;
  g_f4_tile.store(pair ? -cols : cols, std::memory_order_relaxed);
  return CDB_OK;
}

extern "C" int cdb_fp4_gemm(const void* a_v, const void* w_v, const void* bias, void* out, int64_t M, int64_t N, int64_t K,
                            int64_t ld_out, int format, int dtype, int gelu, int32_t* status_word, void* stream) {
  const F4Matrix* a = static_cast<const F4Matrix*>(a_v);
  const F4Matrix* w = static_cast<const F4Matrix*>(w_v);
  if (!a || !w || M < 0 || N <= 0 || K <= 0 || ld_out < N || (format != CDB_NVFP4 && format != CDB_MXFP4) ||
      (dtype != CDB_BF16 && dtype != CDB_F16))
    return CDB_ERR_BAD_ARGUMENT;
  if (M == 0) return CDB_OK;
  const bool nv = format == CDB_NVFP4;
  if (!a->codes || !a->block_scales || !w->codes || !w->block_scales || !out || (nv && (!a->row_scale || !w->row_scale)))
    return CDB_ERR_BAD_ARGUMENT;
  if (K % 32 != 0 || K > FP4_MAX_COLS || N % 8 != 0 || ld_out % 8 != 0 || M > INT32_MAX || N > INT32_MAX ||
      !aligned16(a->codes) || !aligned16(a->block_scales) || !aligned16(w->codes) || !aligned16(w->block_scales) ||
      !aligned16(out))
    return CDB_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CDB_BF16)
    return nv ? f4_gemm<true, __nv_bfloat16>(*a, *w, bias, out, M, N, K, ld_out, gelu, status_word, st)
              : f4_gemm<false, __nv_bfloat16>(*a, *w, bias, out, M, N, K, ld_out, gelu, status_word, st);
  return nv ? f4_gemm<true, __half>(*a, *w, bias, out, M, N, K, ld_out, gelu, status_word, st)
            : f4_gemm<false, __half>(*a, *w, bias, out, M, N, K, ld_out, gelu, status_word, st);
}

// Quantisation and product in one call: the 4-bit form of x lives in the caller's workspace.
extern "C" size_t cdb_fp4_linear_workspace_bytes(int64_t M, int64_t K, int format) {
  if (M <= 0 || K <= 0 || (format != CDB_NVFP4 && format != CDB_MXFP4)) return 0;
  return (size_t)((M * (K / 2) + 255) / 256 * 256) + cdb_fp4_block_scale_bytes(M, K, format) + (size_t)M * 4;
}

extern "C" int cdb_fp4_linear(const void* x, int64_t ld_x, const void* w, const void* bias, void* out, int64_t M, int64_t N,
                              int64_t K, int64_t ld_out, int format, int dtype, int gelu, void* workspace,
                              size_t workspace_bytes, int32_t* status_word, void* stream) {
  if (M == 0) return CDB_OK;
  if (M < 0 || K <= 0 || !workspace) return CDB_ERR_BAD_ARGUMENT;
  if (workspace_bytes < cdb_fp4_linear_workspace_bytes(M, K, format)) return CDB_ERR_SCRATCH_TOO_SMALL;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + (M * (K / 2) + 255) / 256 * 256;
  const bool nv = format == CDB_NVFP4;
  float* row = nv ? reinterpret_cast<float*>(scales + cdb_fp4_block_scale_bytes(M, K, format)) : nullptr;
  const int rc = cdb_fp4_quant_rows(x, M, K, ld_x, dtype, format, codes, scales, row, stream);
  if (rc != CDB_OK) return rc;
  const F4Matrix a{codes, scales, row};
  return cdb_fp4_gemm(&a, w, bias, out, M, N, K, ld_out, format, dtype, gelu, status_word, stream);
}
