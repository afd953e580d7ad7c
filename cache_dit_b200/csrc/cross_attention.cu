// Attention of tokens to an encoder's states of another length:
//
//   out[b, s, h, :] = sum_t softmax_t(scale * q[b, s, h, :] . k[b, t, h / G, :]) v[b, t, h / G, :]   over the kept keys t
//
// G query heads share a key / value head; `key_mask` [batch, keys] names the kept keys.  A batch entry that keeps none
// gives zeros, and what lies in masked places (infinities and NaN too) is never part of a result.
//
// One pass over the keys with a running maximum m and sum l per row (online softmax), on tensor memory:
//   * a CTA per SM takes two tiles of 128 rows, (128 / G) queries x G heads that share a key head, so K and V are read
//     once for the group; work items are spread over a persistent grid, K and V tiles of 128 keys come by TMA into a ring;
//   * S = Q K^T (128 x 128 fp32) in tensor memory; a warpgroup per tile reads its row (a thread per row) and writes
//     P = exp2(S c - m c) in the tensors' type back to tensor memory, from where P V accumulates.  P has columns of its
//     own: as soon as S is read, the next product of scores may overwrite it, and a tile's exponentials run beside the
//     other tile's products.  (With P over S the chain S -> P -> P V -> next S of one tile set the pace, 3600 clocks a
//     step of both tiles; the tensor core needs 2040.)  At d > 64 there is room for one S, which the tiles take in turn;
//   * the output goes through shared memory and TMA: stores of a thread per row took 5500 clocks a tile;
//   * O is rescaled only when a row's maximum has grown by more than 2^8: until then P simply grows to at most 2^8, which
//     costs nothing in a floating type.  P is rounded to 16 bits for the product (a relative 2^-8 or 2^-11 each at most,
//     averaged over the keys); m, l, S and O are fp32.  In fp16, P and l carry a factor of 2^7, the largest that keeps P
//     below 2^16: weights under 2^-25 of the largest would round to zero, and thousands of them may stand beside one key
//     that dominates.  With it a key loses 2^-32 of the largest at most.
// Few rows over many keys: the key range is split over CTAs, partial (O, m, l) are joined by a second kernel.
//
// Warps: 0..3 and 4..7 the tiles' softmax and output, 8 TMA, 9 and 10 the tiles' products.
// Every wait is bounded: on expiry the roles drain, tensor memory is freed and the kernel returns.
#include <cmath>

#include "tcgen05.cuh"

namespace cdb {

constexpr int XA_THREADS = 352;
constexpr int XA_TMA_WARP = 8, XA_MMA_WARP = 9;  // the tiles' products: XA_MMA_WARP + t
constexpr int XA_ROWS = 128;  // rows of a tile
constexpr int XA_KEYS = 128;  // keys of a step
constexpr int XA_MAX_STAGES = 10;
constexpr int XA_MAX_SPLIT = 64;
constexpr int XA_MAX_GROUP = 32;  // heads of a tile
constexpr float XA_LAZY = 8.0f;  // log2 of how far P may grow before O is rescaled
constexpr float XA_F16_RAISE = 7.0f;  // log2 of the factor on P and l in fp16
constexpr int XA_BOX_BYTES = 128 * 128;  // 128 rows x 64 elements
constexpr int XA_WARP_BOX = XA_BOX_BYTES / 4;
template <int DP>
constexpr int xa_tile_bytes() { return XA_BOX_BYTES * (DP / 64); }
template <int DP>
constexpr int xa_stages() { return DP == 128 ? 4 : 10; }
template <int DP>
constexpr int xa_smem() { return 1024 + (2 + xa_stages<DP>()) * xa_tile_bytes<DP>() + 2 * XA_BOX_BYTES + 512; }
// Tensor memory columns: S (one or two) | P0 | P1 | O0 | O1.  With one S the order is P0 S P1 O0 O1.
template <int DP>
constexpr int xa_s_count() { return DP == 64 ? 2 : 1; }
template <int DP>
__host__ __device__ constexpr uint32_t xa_s_col(int t) { return DP == 64 ? 128u * (uint32_t)t : 64u; }
template <int DP>
__host__ __device__ constexpr uint32_t xa_p_col(int t) { return DP == 64 ? 256u + 64u * (uint32_t)t : 192u * (uint32_t)t; }
template <int DP>
__host__ __device__ constexpr uint32_t xa_o_col(int t) { return DP == 64 ? 384u + 64u * (uint32_t)t : 256u + 128u * (uint32_t)t; }
static_assert(xa_smem<128>() <= 232448 && xa_smem<64>() <= 232448, "shared memory");

struct __align__(8) XaBarriers {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[XA_MAX_STAGES], kv_empty[XA_MAX_STAGES];
  uint64_t s_full[2];               // a tile's S is in tensor memory
  uint64_t s_turn[2];               // S is read and a tile's products of scores may overwrite it
  uint64_t p_full[2][2];            // P of a half of the keys written; by an item's first one its predecessor's O is read
  uint64_t pv_done[2];              // a tile's P V complete
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(XaBarriers) <= 512, "barriers");

struct XaParams {
  CUtensorMap map_q, map_k, map_v, map_out;
  void* out;
  float* part_o;    // [splits][rows][D], or null
  float2* part_ml;  // [splits][rows]: (m c, l)
  const uint32_t* words;  // [batch][key_tiles][4] kept keys, or null: all
  const int* list;        // [batch][key_tiles] tiles with a kept key, in order
  const int* count;       // [batch]
  int batch, sq, skv, heads, kv_heads, d;
  int g, q_per_tile, chunks;  // heads of a tile, queries of a tile, tiles per key head's group
  int q_pairs, splits, items, key_tiles;
  float c;  // scale * log2(e)
};

// One work item: two tiles of queries of one head group, over a part of the key tiles.
struct XaItem {
  int b, kv_head, head0, q0, tiles, first, steps, split;
};
__device__ __forceinline__ XaItem xa_item(const XaParams& p, int i) {
  XaItem it;
  it.split = i % p.splits;
  i /= p.splits;
  const int pair = i % p.q_pairs;
  i /= p.q_pairs;
  const int chunk = i % p.chunks;
  i /= p.chunks;
  it.kv_head = i % p.kv_heads;
  it.b = i / p.kv_heads;
  it.head0 = it.kv_head * (p.heads / p.kv_heads) + chunk * p.g;
  it.q0 = pair * 2 * p.q_per_tile;
  it.tiles = p.sq - it.q0 > p.q_per_tile ? 2 : 1;
  const int all = p.count != nullptr ? __ldg(p.count + it.b) : p.key_tiles;
  it.first = (int)((int64_t)all * it.split / p.splits);
  it.steps = (int)((int64_t)all * (it.split + 1) / p.splits) - it.first;
  return it;
}
__device__ __forceinline__ int xa_key_tile(const XaParams& p, const XaItem& it, int j) {
  return p.list != nullptr ? __ldg(p.list + (int64_t)it.b * p.key_tiles + it.first + j) : it.first + j;
}

struct XaRing {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++stage == n) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// tcgen05 instructions of a whole, converged warp: each elects its issuing lane itself (under a branch on an elected lane
// the compiler spends many clocks making each operand uniform).  Loads and stores of tensor memory (.aligned) are the whole
// warp's too, so what depends on the lane is followed by __syncwarp() before them.
#define CDB_XA_ELECTED(text) "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\t" text "\n\t}"
__device__ __forceinline__ void xa_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(CDB_XA_ELECTED("setp.ne.b32 p, %4, 0;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;")
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void xa_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(CDB_XA_ELECTED("setp.ne.b32 p, %4, 0;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;")
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void xa_commit(uint64_t* bar) {
  asm volatile(CDB_XA_ELECTED("@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];")
               ::"r"(smem_u32(bar)) : "memory");
}
// kind::f16: [4,6) D = f32 (1), [7,10) and [10,13) A and B format (0 = f16, 1 = bf16), bit 16 B is N-major, [17,23) N >> 3,
// [24,29) M >> 4.
constexpr uint32_t xa_idesc(bool bf16, int n, bool b_n_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_n_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(XA_ROWS >> 4) << 24);
}
// V as the B operand, N-major: rows of 64 elements (128 bytes, swizzled in groups of 8 rows = 8 keys, 1024 bytes apart);
// the next 64 columns are a box (16 KB) further on.
__device__ __forceinline__ uint64_t xa_v_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(XA_BOX_BYTES >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float xa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float xa_max3(float a, float b, float c) {  // NaN if any is
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t xa_pack(float lo, float hi) {
  if constexpr (__is_same(T, __nv_bfloat16)) {
    return pack_bf16x2(lo, hi);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(XA_THREADS, 1) cross_attention_kernel(const __grid_constant__ XaParams p, int32_t* status_word) {
  constexpr int STAGES = xa_stages<DP>();
  constexpr int TILE = xa_tile_bytes<DP>();
  constexpr int BOXES = DP / 64;
  constexpr bool BF16 = __is_same(T, __nv_bfloat16);
  constexpr float NEG_INF = -INFINITY;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;
  uint8_t* s_kv = smem + 2 * TILE;
  uint8_t* s_out = s_kv + STAGES * TILE;  // 32 rows x 64 columns of output per softmax warp
  XaBarriers* gb = reinterpret_cast<XaBarriers*>(s_out + 2 * XA_BOX_BYTES);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&gb->q_full[t], 1);
      mbar_init(&gb->q_empty[t], 1);
      mbar_init(&gb->s_full[t], 1);
      mbar_init(&gb->p_full[t][0], 4);
      mbar_init(&gb->p_full[t][1], 4);
      mbar_init(&gb->s_turn[t], 4);
      mbar_init(&gb->pv_done[t], 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&gb->kv_full[s], 1);
      mbar_init(&gb->kv_empty[s], 2);
    }
    gb->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == XA_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&gb->tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, gb->tmem_base, 0);
  pdl_wait_prior();  // the mask kernel's words, and the producers of q, k, v

  if (warp == XA_TMA_WARP) {
    // ---------------- loads ----------------
    if (lane == 0) {
      XaRing at;
      uint32_t issued = 0, q_uses = 0, q_used = 0;  // bit t: phase of the tile's next Q, and whether it had one
      bool ok = true;
      const uint32_t q_tx = (uint32_t)(p.g * p.q_per_tile * 128 * BOXES);
      for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
        const XaItem it = xa_item(p, i);
        if (it.steps == 0) continue;
        for (int j = 0; j < it.steps && ok; ++j) {
          const int key0 = xa_key_tile(p, it, j) * XA_KEYS;
          if (j == 0) {
            for (int t = 0; t < it.tiles && ok; ++t) {
              ok = bounded_wait(&gb->q_empty[t], ((q_uses >> t) & 1u) ^ 1u, &gb->abort_flag, status_word, 31);
              if (!ok) break;
              q_uses ^= 1u << t;
              q_used |= 1u << t;
              mbar_expect_tx(&gb->q_full[t], q_tx);
              for (int x = 0; x < BOXES; ++x)
                tma_load_4d(&p.map_q, &gb->q_full[t], s_q + t * TILE + x * XA_BOX_BYTES, x * 64, it.head0,
                            it.q0 + t * p.q_per_tile, it.b);
            }
            if (!ok) break;
          }
          for (int kv = 0; kv < 2 && ok; ++kv) {
            ok = bounded_wait(&gb->kv_empty[at.stage], at.phase ^ 1u, &gb->abort_flag, status_word, 32);
            if (!ok) break;
            mbar_expect_tx(&gb->kv_full[at.stage], TILE);
            for (int x = 0; x < BOXES; ++x)
              tma_load_4d(kv ? &p.map_v : &p.map_k, &gb->kv_full[at.stage], s_kv + at.stage * TILE + x * XA_BOX_BYTES, x * 64,
                          it.kv_head, key0, it.b);
            at.next(STAGES);
            ++issued;
          }
        }
      }
      // The CTA may not retire while copies into its shared memory are in flight, while MMAs read it or while a commit has
      // yet to arrive on one of its barriers: wait (bounded, also after an abort) until the MMAs released every stage and Q
      // used, the last commits that are issued.  (The last P V's own commit comes before that of its stage.)
      const uint64_t t0 = global_timer_ns();
      for (uint32_t j = issued > (uint32_t)STAGES ? issued - STAGES : 0; j < issued; ++j)
        while (!mbar_try_wait(&gb->kv_empty[j % STAGES], (j / STAGES) & 1u) && global_timer_ns() - t0 < BARRIER_LIMIT_NS) {}
      for (int t = 0; t < 2; ++t)
        while (((q_used >> t) & 1u) && !mbar_try_wait(&gb->q_empty[t], ((q_uses >> t) & 1u) ^ 1u) && global_timer_ns() - t0 < BARRIER_LIMIT_NS) {}
    }
    __syncwarp();
  } else if (warp >= XA_MMA_WARP) {
    // ---------------- products of tile t ----------------
    // For every step: S = Q_t K^T, then O_t += P_t V of the step before, whose exponentials ran meanwhile.  A warp per
    // tile: a satisfied wait takes 60 to 100 clocks, and one warp that did them all for both tiles set the pace.
    const int t = warp - XA_MMA_WARP;
    constexpr uint32_t idesc_s = xa_idesc(BF16, XA_KEYS, false);
    constexpr uint32_t idesc_o = xa_idesc(BF16, DP, true);
    const uint32_t q_base = smem_u32(s_q) + t * TILE;
    const uint32_t kv_base = smem_u32(s_kv);
    const uint32_t s_addr = tmem_base + (t ? xa_s_col<DP>(1) : xa_s_col<DP>(0));
    const uint32_t p_addr = tmem_base + (t ? xa_p_col<DP>(1) : xa_p_col<DP>(0));
    const uint32_t o_addr = tmem_base + (t ? xa_o_col<DP>(1) : xa_o_col<DP>(0));
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
      return warp_wait(bar, phase, &gb->abort_flag, status_word, code);
    };
    bool due = false, due_first = false;  // a P V to be issued
    int due_stage = 0;
    uint32_t due_phase = 0;
    XaRing at;  // K of the current step; V follows it
    uint32_t p_uses = 0, q_uses = 0, turns = 0;
    bool ok = true;
    auto values = [&] {  // O_t += P_t V
      ok = wait(&gb->kv_full[due_stage], due_phase, 35);
      const uint64_t v = xa_v_desc(kv_base + due_stage * TILE);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (ok) ok = wait(&gb->p_full[t][half], p_uses & 1u, 36);
        if (!ok) return;
        tcgen05_fence_after();
#pragma unroll
        for (int k = half * 4; k < half * 4 + 4; ++k)  // 16 keys: 8 columns of P, 2048 bytes of V
          xa_mma_ts(o_addr, p_addr + k * 8, v + (uint64_t)(k * (2048 >> 4)), idesc_o, !due_first || k != 0);
      }
      xa_commit(&gb->pv_done[t]);
      xa_commit(&gb->kv_empty[due_stage]);
      ++p_uses;
      due = false;
    };
    // After the last item one more round without scores: it issues what is outstanding.
    for (int i = blockIdx.x; ok && (i < p.items || due); i += gridDim.x) {
      XaItem it{};
      if (i < p.items) it = xa_item(p, i);
      if (i >= p.items || (t >= it.tiles && it.steps > 0)) {
        if (due) values();
        if (!ok) break;
      }
      for (int j = 0; j < it.steps && ok; ++j) {
        const int k_stage = at.stage;
        ok = wait(&gb->kv_full[k_stage], at.phase, 33);
        if (!ok) break;
        at.next(STAGES);
        if (t >= it.tiles) {  // the other tile's alone: K and V are released for this one
          if (lane == 0) mbar_arrive(&gb->kv_empty[k_stage]);
          ok = wait(&gb->kv_full[at.stage], at.phase, 38);
          if (!ok) break;
          if (lane == 0) mbar_arrive(&gb->kv_empty[at.stage]);
          at.next(STAGES);
          continue;
        }
        if (j == 0) {
          ok = wait(&gb->q_full[t], q_uses & 1u, 34);
          if (!ok) break;
          ++q_uses;
        }
        // Two S: this tile's last one is read.  One S: the tiles take turns, and who read the last one passes the turn on;
        // so every phase of a turn belongs to one product.  The first product of all finds S free.
        ok = wait(&gb->s_turn[t], (turns & 1u) ^ (DP == 64 || t == 0 ? 1u : 0u), 37);
        if (!ok) break;
        ++turns;
        tcgen05_fence_after();
        const uint64_t a = make_kmajor_sw128_desc(q_base), b = make_kmajor_sw128_desc(kv_base + k_stage * TILE);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {  // 16 elements = 32 bytes; a box holds 64
          const uint64_t off = (uint64_t)((k / 4) * (XA_BOX_BYTES >> 4) + (k % 4) * 2);
          xa_mma_ss(s_addr, a + off, b + off, idesc_s, k != 0);
        }
        xa_commit(&gb->s_full[t]);
        if (j + 1 == it.steps) xa_commit(&gb->q_empty[t]);
        xa_commit(&gb->kv_empty[k_stage]);
        if (due) values();
        due = true;
        due_first = j == 0;
        due_stage = at.stage;
        due_phase = at.phase;
        at.next(STAGES);
      }
    }
    __syncwarp();
  } else {
    // ---------------- softmax and output of tile t: a thread per row ----------------
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem_base + lanes + (t ? xa_s_col<DP>(1) : xa_s_col<DP>(0));
    const uint32_t p_addr = tmem_base + lanes + (t ? xa_p_col<DP>(1) : xa_p_col<DP>(0));
    const uint32_t o_addr = tmem_base + lanes + (t ? xa_o_col<DP>(1) : xa_o_col<DP>(0));
    XaRing at;  // follows the ring of K and V tiles where there is a mask
    uint32_t s_uses = 0;
    bool ok = true;
    // What the last item's output needs; it is written once its last P V is complete, while the next one's scores wait.
    bool pending = false;
    int out_b = 0, out_q0 = 0, out_head0 = 0;
    int64_t out_row = -1;   // row of `out`, -1: none (beyond the last query, or a row of no head)
    int64_t part_base = 0;  // first row of the split's partial results
    float m = 0.f, l = 0.f;
    auto write_out = [&] {
      pending = false;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
      if (p.part_o != nullptr) {
        float* dst = p.part_o + (part_base + out_row) * p.d;
#pragma unroll 1
        for (int c0 = 0; c0 < DP && c0 < p.d; c0 += 16) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(o_addr + c0, o);
          tmem_ld_wait();
          if (out_row >= 0) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (c0 + 4 * x < p.d) *reinterpret_cast<uint4*>(dst + c0 + 4 * x) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
          __syncwarp();  // the next load from tensor memory is the whole warp's
        }
        if (out_row >= 0) p.part_ml[part_base + out_row] = make_float2(m == NEG_INF ? 0.f : m * p.c, l);
      } else {
        // This warp's 32 rows, 64 columns at a time, through shared memory (128-byte rows, swizzled as the tensor map has
        // it); the copy out clips queries and columns that do not exist.
        uint8_t* box = s_out + warp * XA_WARP_BOX;
#pragma unroll 1
        for (int x = 0; x < BOXES; ++x) {
          if (lane == 0) bulk_wait_group_read<0>();  // the copy before this one has read the buffer
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_addr + x * 64 + h * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t w[4];
#pragma unroll
              for (int z = 0; z < 4; ++z)
                w[z] = xa_pack<T>(__uint_as_float(o[8 * y + 2 * z]) * inv, __uint_as_float(o[8 * y + 2 * z + 1]) * inv);
              *reinterpret_cast<uint4*>(box + lane * 128 + (((h * 2 + y) ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (out_q0 < p.sq) tma_store_4d(&p.map_out, box, x * 64, out_head0, out_q0, out_b);
            bulk_commit_group();
          }
        }
      }
      __syncwarp();
    };
    uint32_t posted = 0;
    // The tile's last P V is complete: its P may be overwritten, its O read.
    auto values_done = [&] {
      return posted == 0 || warp_wait(&gb->pv_done[t], (posted - 1) & 1u, &gb->abort_flag, status_word, 42);
    };
    for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const XaItem it = xa_item(p, i);
      const int qi = row / p.g, h = row - qi * p.g;
      const int s = it.q0 + t * p.q_per_tile + qi;
      const int64_t next_row = qi < p.q_per_tile && s < p.sq ? ((int64_t)it.b * p.sq + s) * p.heads + it.head0 + h : -1;
      const int64_t next_base = (int64_t)it.split * p.batch * p.sq * p.heads;
      if (t >= it.tiles) {
        for (int j = 0; j < 2 * it.steps; ++j) at.next(STAGES);
        continue;
      }
      if (it.steps == 0) {  // no key is kept: zeros (or an empty part)
        if (next_row >= 0) {
          if (p.part_o != nullptr) {
            for (int x = 0; x < p.d; x += 4) *reinterpret_cast<uint4*>(p.part_o + (next_base + next_row) * p.d + x) = make_uint4(0, 0, 0, 0);
            p.part_ml[next_base + next_row] = make_float2(0.f, 0.f);
          } else {
            for (int x = 0; x < p.d; x += 8) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + next_row * p.d + x) = make_uint4(0, 0, 0, 0);
          }
        }
        __syncwarp();
        continue;
      }
      for (int j = 0; j < it.steps; ++j) {
        const int tile = xa_key_tile(p, it, j);
        uint4 w = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (p.words != nullptr) {
          w = __ldg(reinterpret_cast<const uint4*>(p.words) + (int64_t)it.b * p.key_tiles + tile);
        } else if ((tile + 1) * XA_KEYS > p.skv) {
          const int left = p.skv - tile * XA_KEYS;  // 1..127
          auto bits = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
          w = make_uint4(bits(left), bits(left - 32), bits(left - 64), bits(left - 96));
        }
        ok = warp_wait(&gb->s_full[t], s_uses & 1u, &gb->abort_flag, status_word, 41);
        if (!ok) break;
        ++s_uses;
        tcgen05_fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_32x32b_x32(s_addr + q * 32, v[q]);
        if (p.words != nullptr) {
          // Rows of V that the mask leaves out become zero: 0 * NaN would not be 0.  A thread per key; both tiles do it, each
          // before its own P is posted, so that neither's product can be ahead.
          at.next(STAGES);  // K
          if ((w.x & w.y & w.z & w.w) != 0xffffffffu) {
            ok = warp_wait(&gb->kv_full[at.stage], at.phase, &gb->abort_flag, status_word, 40);
            if (!ok) break;
            const uint32_t word = (warp & 2) ? ((warp & 1) ? w.w : w.z) : ((warp & 1) ? w.y : w.x);
            if (!((word >> lane) & 1u)) {
              uint4* v_row = reinterpret_cast<uint4*>(s_kv + at.stage * TILE + row * 128);  // 128 bytes in each box
#pragma unroll
              for (int x = 0; x < BOXES; ++x)
#pragma unroll
                for (int y = 0; y < 8; ++y) v_row[x * (XA_BOX_BYTES / 16) + y] = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
            __syncwarp();
          }
          at.next(STAGES);  // V
        }
        tmem_ld_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&gb->s_turn[DP == 64 ? t : (t == 0 && it.tiles == 2 ? 1 : 0)]);  // the next scores may overwrite S
        __syncwarp();
        if ((w.x & w.y & w.z & w.w) != 0xffffffffu) {
          const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int x = 0; x < 32; ++x) v[q][x] = (word[q] >> x) & 1u ? v[q][x] : 0xff800000u;
        }
        float top4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top4[q] = xa_max3(__uint_as_float(v[q][0]), __uint_as_float(v[q][1]), __uint_as_float(v[q][2]));
#pragma unroll
          for (int x = 3; x < 31; x += 2) top4[q] = xa_max3(top4[q], __uint_as_float(v[q][x]), __uint_as_float(v[q][x + 1]));
          top4[q] = xa_max3(top4[q], top4[q], __uint_as_float(v[q][31]));
        }
        const float top = xa_max3(xa_max3(top4[0], top4[1], top4[2]), top4[3], top4[3]);
        ok = values_done();
        if (!ok) break;
        tcgen05_fence_after();
        if (pending) write_out();
        if (j == 0) {
          m = top;
          l = 0.f;
        } else if (__any_sync(0xffffffffu, !((top - m) * p.c <= XA_LAZY))) {  // a NaN too
          const float grown = xa_max3(m, top, top);
          const float f = m == NEG_INF ? 0.f : xa_exp2((m - grown) * p.c);
          m = grown;
          l *= f;
#pragma unroll 1
          for (int c0 = 0; c0 < DP; c0 += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_addr + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st_32x32b_x16(o_addr + c0, o);
          }
          tmem_st_wait();
        }
        const float mc = m == NEG_INF ? 0.f : m * p.c - (BF16 ? 0.f : XA_F16_RAISE);  // a row of -inf alone: P = 0
        const uint64_t c2 = f32_pair(p.c, p.c), mc2 = f32_pair(-mc, -mc);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            uint64_t e = f32_fma2(f32_pair(__uint_as_float(v[q][2 * x]), __uint_as_float(v[q][2 * x + 1])), c2, mc2);
            float lo, hi;
            f32_unpair(e, lo, hi);
            lo = xa_exp2(lo);
            hi = xa_exp2(hi);
            sum2[x & 1] = f32_add2(sum2[x & 1], f32_pair(lo, hi));
            pk[x] = xa_pack<T>(lo, hi);
          }
          tmem_st_32x32b_x16(p_addr + q * 16, pk);
          if (q & 1) {  // the products over these 64 keys may start
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&gb->p_full[t][q >> 1]);
            __syncwarp();
          }
        }
        float l0, l1;
        f32_unpair(f32_add2(sum2[0], sum2[1]), l0, l1);
        l += l0 + l1;
        ++posted;
      }
      if (!ok) break;
      pending = true;
      out_row = next_row;
      part_base = next_base;
      out_b = it.b;
      out_q0 = it.q0 + t * p.q_per_tile + (warp & 3) * (p.q_per_tile / 4);
      out_head0 = it.head0;
    }
    if (ok && pending && values_done()) {
      tcgen05_fence_after();
      write_out();
    }
    if (lane == 0) bulk_wait_group_all();  // the output is written before the CTA retires
    __syncwarp();
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == XA_MMA_WARP) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// Kept keys as bits, and the tiles of 128 keys that keep any, in order.  A CTA per batch entry, a warp per tile.
__global__ void __launch_bounds__(1024)
    cross_mask_kernel(const uint8_t* __restrict__ mask, int64_t ld_mask, int skv, int key_tiles, uint32_t* __restrict__ words,
                      int* __restrict__ list, int* __restrict__ count) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint8_t* row = mask + (int64_t)b * ld_mask;
  uint4* w4 = reinterpret_cast<uint4*>(words) + (int64_t)b * key_tiles;
  for (int tile = warp; tile < key_tiles; tile += 32) {
    uint32_t keep[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int key = tile * XA_KEYS + q * 32 + lane;
      keep[q] = key < skv ? row[key] : 0;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) keep[q] = __ballot_sync(0xffffffffu, keep[q] != 0);
    if (lane == 0) w4[tile] = make_uint4(keep[0], keep[1], keep[2], keep[3]);
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int base = 0; base < key_tiles; base += 32) {
      const int tile = base + lane;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (tile < key_tiles) w = w4[tile];
      const uint32_t any = __ballot_sync(0xffffffffu, (w.x | w.y | w.z | w.w) != 0u);
      if (any >> lane & 1u) list[(int64_t)b * key_tiles + n + __popc(any & ((1u << lane) - 1u))] = tile;
      n += __popc(any);
    }
    if (lane == 0) count[b] = n;
  }
}

// Joins the parts of a split key range: a warp per row, four columns per lane.
template <typename T>
__global__ void __launch_bounds__(256)
    cross_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* __restrict__ out, int64_t rows,
                      int splits, int d) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x & 31;
  for (int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5; row < rows; row += (int64_t)gridDim.x * 8) {
    float2 ml[XA_MAX_SPLIT / 32];
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < XA_MAX_SPLIT / 32; ++q) {
      const int s = q * 32 + lane;
      ml[q] = s < splits ? part_ml[(int64_t)s * rows + row] : make_float2(0.f, 0.f);
      if (ml[q].y != 0.f) top = fmaxf(top, ml[q].x);
    }
    top = warp_max(top);
    float total = 0.f;
#pragma unroll
    for (int q = 0; q < XA_MAX_SPLIT / 32; ++q) {
      ml[q].x = ml[q].y != 0.f ? exp2f(ml[q].x - top) : 0.f;  // the part's weight
      total = fmaf(ml[q].x, ml[q].y, total);
    }
    total = warp_sum(total);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int c = lane * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < XA_MAX_SPLIT / 32; ++q) {
      for (int s = q * 32; s < min(splits, q * 32 + 32); ++s) {
        const float f = __shfl_sync(0xffffffffu, ml[q].x, s & 31);
        if (c < d && f != 0.f) {
          const float4 o = __ldcs(reinterpret_cast<const float4*>(part_o + ((int64_t)s * rows + row) * d + c));
          acc.x = fmaf(f, o.x, acc.x);
          acc.y = fmaf(f, o.y, acc.y);
          acc.z = fmaf(f, o.z, acc.z);
          acc.w = fmaf(f, o.w, acc.w);
        }
      }
    }
    if (c < d)
      *reinterpret_cast<uint2*>(out + row * d + c) = make_uint2(xa_pack<T>(acc.x * inv, acc.y * inv), xa_pack<T>(acc.z * inv, acc.w * inv));
  }
}

// ---- host side -----------------------------------------------------------------------------------------------
struct XaPlan {
  int g, q_per_tile, chunks, q_pairs, key_tiles, splits;
  int64_t items, rows;
  size_t words_at, list_at, count_at, ml_at, o_at, bytes;  // workspace
};
static size_t xa_round(size_t n) { return (n + 255) / 256 * 256; }

// Heads of a tile: the largest power of two up to 32 that divides the group, so that 32 rows, a warp's, are whole
// queries of all of them.  Splits of the key range: items cost their steps plus about four more for their first loads
// and their output; a split launch about four for the join, and the time its fp32 partials take to HBM and back, a step
// (1.4 to 1.6 us) for 8.5 MB.  The number of splits is the one whose waves over the SMs cost least.  Measured, unsplit
// against the best split: 1 x 6400 x 4096, 12 heads of 128 175 : 218 us (2 parts), 1 x 1024 x 4096 x 24 65 : 75 (3),
// 1 x 256 x 1024 x 40 20 : 25 (2), 1 x 300 x 4096 x 24 59 : 37 (3), 1 x 2560 x 8192 x 15 224 : 206 (3; 2 and 4 parts 208
// and 210), one query on 16385 keys, 4 x 32 heads on 8 key heads 193 : 59 (4).
static XaPlan xa_plan(int64_t batch, int64_t sq, int64_t skv, int64_t heads, int64_t kv_heads, int64_t d, bool masked, int sms) {
  XaPlan p{};
  const int group = (int)(heads / kv_heads);
  for (p.g = 1; p.g < XA_MAX_GROUP && group % (2 * p.g) == 0;) p.g *= 2;
  p.q_per_tile = XA_ROWS / p.g;
  p.chunks = group / p.g;
  p.q_pairs = (int)((sq + 2 * p.q_per_tile - 1) / (2 * p.q_per_tile));
  p.key_tiles = (int)((skv + XA_KEYS - 1) / XA_KEYS);
  p.rows = batch * sq * heads;
  const int64_t items = batch * kv_heads * p.chunks * p.q_pairs;
  p.splits = 1;
  double best = 1e300;
  for (int n = 1; n <= XA_MAX_SPLIT && n <= p.key_tiles; ++n) {
    const int64_t waves = (items * n + sms - 1) / sms;
    const double partials = n > 1 ? 2.0 * n * (double)p.rows * (double)(d * 4 + 8) : 0.0;  // bytes, written and read
    const double cost = (double)waves * ((p.key_tiles + n - 1) / n + 4) + (n > 1 ? 4 : 0) + partials / 8.5e6;
    if (cost < best) {
      best = cost;
      p.splits = n;
    }
  }
  p.items = items * p.splits;
  size_t at = 0;
  if (masked) {
    p.words_at = at;
    at += xa_round((size_t)batch * p.key_tiles * 16);
    p.list_at = at;
    at += xa_round((size_t)batch * p.key_tiles * 4);
    p.count_at = at;
    at += xa_round((size_t)batch * 4);
  }
  if (p.splits > 1) {
    p.ml_at = at;
    at += xa_round((size_t)p.splits * p.rows * 8);
    p.o_at = at;
    at += xa_round((size_t)p.splits * p.rows * d * 4);
  }
  p.bytes = at;
  return p;
}

static bool xa_map(CUtensorMap* map, bool bf16, const cdb_heads& t, int64_t d, int64_t heads, int64_t tokens, int64_t batch,
                   int box_heads, int box_tokens) {
  const EncodeTiledFn fn = tensor_map_encoder();
  // a dimension of extent 1 is never stepped over: any legal stride will do
  auto stride = [](int64_t elements, int64_t extent) { return (cuuint64_t)(extent > 1 ? elements * 2 : 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {stride(t.head_stride, heads), stride(t.token_stride, tokens), stride(t.batch_stride, batch)};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens, 1}, ones[4] = {1, 1, 1, 1};
  return fn != nullptr && fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                             const_cast<void*>(t.data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
static int xa_launch(const XaParams& prm, int sms, int32_t* status_word, cudaStream_t st) {
  static PerDevice attr_state;
  const cudaError_t attr_err = (cudaError_t)attr_state.get([]() -> int64_t {
    return (int64_t)cudaFuncSetAttribute(cross_attention_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, xa_smem<DP>());
  });
  CDB_CUDA_CHECK(attr_err);
  const unsigned grid = (unsigned)(prm.items < sms ? prm.items : sms);
  CDB_CUDA_CHECK(launch_pdl(cross_attention_kernel<T, DP>, dim3(grid), dim3(XA_THREADS), (size_t)xa_smem<DP>(), st, prm, status_word));
  return CDB_OK;
}

static bool xa_sizes_ok(int64_t batch, int64_t sq, int64_t skv, int64_t heads, int64_t kv_heads, int64_t d) {
  return batch >= 0 && sq >= 0 && skv >= 0 && heads > 0 && kv_heads > 0 && d > 0 && heads % kv_heads == 0;
}
static bool xa_strides_ok(const cdb_heads& t, int64_t heads, int64_t tokens, int64_t batch) {
  // a tensor map's strides: multiples of 16 bytes, below 2^40
  auto ok = [](int64_t s, int64_t extent) { return extent <= 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
  return aligned16(t.data) && ok(t.head_stride, heads) && ok(t.token_stride, tokens) && ok(t.batch_stride, batch);
}

}  // namespace cdb

using namespace cdb;

extern "C" size_t cdb_cross_attention_workspace_bytes(int64_t batch, int64_t sq, int64_t skv, int64_t heads, int64_t kv_heads,
                                                      int64_t d, int masked) {
  if (!xa_sizes_ok(batch, sq, skv, heads, kv_heads, d) || batch == 0 || sq == 0 || skv == 0) return 0;
  return xa_plan(batch, sq, skv, heads, kv_heads, d, masked != 0, sm_count()).bytes;
}

extern "C" int cdb_cross_attention(const void* q_v, const void* k_v, const void* v_v, const void* key_mask, int64_t ld_mask,
                                   void* out, int64_t batch, int64_t sq, int64_t skv, int64_t heads, int64_t kv_heads, int64_t d,
                                   float scale, int dtype, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                   void* stream) {
  const cdb_heads* q = static_cast<const cdb_heads*>(q_v);
  const cdb_heads* k = static_cast<const cdb_heads*>(k_v);
  const cdb_heads* v = static_cast<const cdb_heads*>(v_v);
  if (!q || !k || !v || !xa_sizes_ok(batch, sq, skv, heads, kv_heads, d) || (dtype != CDB_BF16 && dtype != CDB_F16) ||
      !(scale > 0.f) || !std::isfinite(scale))
    return CDB_ERR_BAD_ARGUMENT;
  if (batch == 0 || sq == 0) return CDB_OK;
  if (!out || !q->data || (skv > 0 && (!k->data || !v->data))) return CDB_ERR_BAD_ARGUMENT;
  if (d > CDB_CROSS_MAX_HEAD_DIM || d % 8 != 0 || !aligned16(out)) return CDB_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (skv == 0) {  // nothing to attend to
    CDB_CUDA_CHECK(cudaMemsetAsync(out, 0, (size_t)batch * sq * heads * d * 2, st));
    return CDB_OK;
  }
  if (!xa_strides_ok(*q, heads, sq, batch) || !xa_strides_ok(*k, kv_heads, skv, batch) || !xa_strides_ok(*v, kv_heads, skv, batch))
    return CDB_ERR_UNSUPPORTED;
  if (sq > INT32_MAX - 256 || skv > INT32_MAX - 256 || heads > 65535 || batch > INT32_MAX) return CDB_ERR_TOO_LARGE;
  const int sms = sm_count();
  const XaPlan plan = xa_plan(batch, sq, skv, heads, kv_heads, d, key_mask != nullptr, sms);
  if (plan.items > INT32_MAX - sms) return CDB_ERR_TOO_LARGE;  // a block's item index goes a grid's step past the last
  if (plan.bytes > workspace_bytes || (plan.bytes > 0 && !workspace)) return CDB_ERR_SCRATCH_TOO_SMALL;
  if (!aligned16(workspace)) return CDB_ERR_UNSUPPORTED;
  const bool bf16 = dtype == CDB_BF16;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  XaParams p{};
  if (!xa_map(&p.map_q, bf16, *q, d, heads, sq, batch, plan.g, plan.q_per_tile) ||
      !xa_map(&p.map_out, bf16, cdb_heads{out, sq * heads * d, heads * d, d}, d, heads, sq, batch, plan.g, plan.q_per_tile / 4) ||
      !xa_map(&p.map_k, bf16, *k, d, kv_heads, skv, batch, 1, XA_KEYS) || !xa_map(&p.map_v, bf16, *v, d, kv_heads, skv, batch, 1, XA_KEYS)) {
    set_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled");
    return CDB_ERR_CUDA;
  }
  p.out = out;
  if (plan.splits > 1) {
    p.part_ml = reinterpret_cast<float2*>(ws + plan.ml_at);
    p.part_o = reinterpret_cast<float*>(ws + plan.o_at);
  }
  if (key_mask != nullptr) {
    uint32_t* words = reinterpret_cast<uint32_t*>(ws + plan.words_at);
    int* list = reinterpret_cast<int*>(ws + plan.list_at);
    int* count = reinterpret_cast<int*>(ws + plan.count_at);
    CDB_CUDA_CHECK(launch_pdl(cross_mask_kernel, dim3((unsigned)batch), dim3(1024), 0, st, static_cast<const uint8_t*>(key_mask),
                              ld_mask, (int)skv, plan.key_tiles, words, list, count));
    p.words = words;
    p.list = list;
    p.count = count;
  }
  p.batch = (int)batch; p.sq = (int)sq; p.skv = (int)skv; p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.d = (int)d;
  p.g = plan.g; p.q_per_tile = plan.q_per_tile; p.chunks = plan.chunks; p.q_pairs = plan.q_pairs; p.splits = plan.splits;
  p.items = (int)plan.items; p.key_tiles = plan.key_tiles;
  p.c = scale * 1.4426950408889634f;
  int rc;
  if (d <= 64) rc = bf16 ? xa_launch<__nv_bfloat16, 64>(p, sms, status_word, st) : xa_launch<__half, 64>(p, sms, status_word, st);
  else rc = bf16 ? xa_launch<__nv_bfloat16, 128>(p, sms, status_word, st) : xa_launch<__half, 128>(p, sms, status_word, st);
  if (rc != CDB_OK || plan.splits == 1) return rc;
  const int64_t want = (plan.rows + 7) / 8, cap = (int64_t)sms * 8;
  const dim3 grid((unsigned)(want < cap ? want : cap));
  if (bf16)
    CDB_CUDA_CHECK(launch_pdl(cross_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p.part_o, p.part_ml,
                              static_cast<__nv_bfloat16*>(out), plan.rows, plan.splits, (int)d));
  else
    CDB_CUDA_CHECK(launch_pdl(cross_join_kernel<__half>, grid, dim3(256), 0, st, p.part_o, p.part_ml, static_cast<__half*>(out),
                              plan.rows, plan.splits, (int)d));
  return CDB_OK;
}
