// Gated residual with a norm on either side, in one pass over the rows:
//
//   x' = x + residual_scale * gate * post(y)          post: none, RMSNorm or LayerNorm of the branch
//   h  = norm(x') * weight + bias, then * (1 + scale) + shift
//
// x' and h are written in the tensors' type, or h in 4 bits for the linear that reads it (fp4.cuh).  Everything between
// is fp32: x' is rounded once where it is stored, and the norm reads the unrounded value; h is rounded to the tensors'
// type before it is quantised, so that the 4-bit form is the quantisation of exactly what the 16-bit form returns.
//
// HBM-bound: x, y in, x', h out.  A row is held in registers by 32 to 256 threads (packs of 8 elements, pack p at
// thread p % threads), so each input byte is read once; statistics are two-pass (mean, then squared deviations), which
// loses nothing to cancellation.
#include "fp4.cuh"

namespace cdb {

constexpr int NORM_THREADS = 256;
enum NormKind { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

struct NormArgs {
  const void *x, *y, *gate, *post_weight, *post_bias, *weight, *bias, *scale, *shift;
  int64_t x_batch, x_row, y_batch, y_row;             // strides in elements
  int64_t gate_batch, scale_batch, shift_batch;       // 0: one vector for all batches
  void *x_out, *h_out;                                // contiguous rows; null: not wanted
  uint8_t *codes, *block_scales;                      // 4-bit h
  float* row_scales;
  int64_t rows;
  int tokens, dim, post, norm, format;                // format: CDB_NVFP4, CDB_MXFP4, or -1 for h_out
  float residual_scale, post_eps, eps;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }  // round to nearest even

// Eight 16-bit elements of a 16-byte packet.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, __nv_bfloat16)) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}
// Which eight elements of a row pack `i` of thread `t` is: eight in a row, as 16-byte accesses, where rows allow it; else
// TPR apart, so that neighbouring threads still touch neighbouring elements (eight in a row, one by one: 154 us for
// 30000 x 1001 bf16).
template <int TPR, bool ALIGNED>
__device__ __forceinline__ int first_column(int t, int i) {
  return ALIGNED ? (t + i * TPR) * 8 : i * 8 * TPR + t;
}
// The eight elements from p on; `n` columns are left in the row (what is beyond reads as 0 and is not written).
template <typename T, bool ALIGNED, int TPR>
__device__ __forceinline__ void load8(const T* p, int n, float (&f)[8]) {
  if constexpr (ALIGNED) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i * TPR < n ? to_f(p[i * TPR]) : 0.f;
  }
}
template <typename T, bool ALIGNED, int TPR>
__device__ __forceinline__ void store8(T* p, int n, const float (&f)[8]) {
  if constexpr (ALIGNED) {
    if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
      __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(T, __nv_bfloat16)) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * TPR < n) p[i * TPR] = from_f<T>(f[i]);
  }
}

// Rounds eight numbers to T and returns the largest magnitude's bits (as integers: infinity and NaN are above all).
template <typename T>
__device__ __forceinline__ uint32_t round8(float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
    return top;
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, __nv_bfloat16)) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    unpack8<T>(make_uint4(w[0], w[1], w[2], w[3]), f);
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    const uint32_t top = max(m & 0xffffu, m >> 16);
    if constexpr (__is_same(T, __nv_bfloat16)) return top << 16;
    else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  }
}

// v = a * b + c and friends on eight numbers, two per instruction.
__device__ __forceinline__ void fma8(float (&v)[8], const float (&a)[8], const float (&b)[8], const float (&c)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    f32_unpair(f32_fma2(f32_pair(a[j], a[j + 1]), f32_pair(b[j], b[j + 1]), f32_pair(c[j], c[j + 1])), v[j], v[j + 1]);
}
__device__ __forceinline__ void mul8(float (&v)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) f32_unpair(f32_mul2(f32_pair(a[j], a[j + 1]), f32_pair(b[j], b[j + 1])), v[j], v[j + 1]);
}
__device__ __forceinline__ void add8(float (&v)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) f32_unpair(f32_add2(f32_pair(a[j], a[j + 1]), f32_pair(b[j], b[j + 1])), v[j], v[j + 1]);
}
__device__ __forceinline__ void fill8(float (&v)[8], float x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x;
}

// Sum (or maximum) over the TPR threads of a row.  `slot` is this reduction's number within the row and the row's
// parity: a warp that is ahead writes other words than the ones a slower warp still reads, and cannot be two rows ahead.
template <int TPR>
__device__ __forceinline__ void row_barrier() {
  __syncwarp();  // the barrier counts whole warps, and a lane that wrote a word may be apart
  asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / TPR), "n"(TPR) : "memory");
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* words) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = v;
    row_barrier<TPR>();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) v += words[(threadIdx.x / TPR) * (TPR / 32) + w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* words) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = __uint_as_float(v);
    row_barrier<TPR>();
    v = 0u;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) v = max(v, __float_as_uint(words[(threadIdx.x / TPR) * (TPR / 32) + w]));
  }
  return v;
}

// The statistics of a row held as v[PACKS][8]: subtracts the mean (LayerNorm) and returns 1 / sqrt(mean square + eps).
template <int TPR, int PACKS, bool ALIGNED>
__device__ __forceinline__ float normalise(float (&v)[PACKS][8], int kind, int t, int dim, float eps, float (*words)[NORM_THREADS / 32]) {
  const float inv_dim = 1.0f / (float)dim;
  if (kind == NORM_LAYER) {
    uint64_t s2[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
      for (int j = 0; j < 8; j += 2) s2[(j >> 1) & 1] = f32_add2(s2[(j >> 1) & 1], f32_pair(v[i][j], v[i][j + 1]));
    float lo, hi;
    f32_unpair(f32_add2(s2[0], s2[1]), lo, hi);
    const float mean = row_sum<TPR>(lo + hi, words[0]) * inv_dim;
    float minus[8];
    fill8(minus, -mean);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int left = dim - first_column<TPR, ALIGNED>(t, i);
      if constexpr (ALIGNED) {  // a pack is all there or not at all
        if (left > 0) add8(v[i], v[i], minus);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = j * TPR < left ? v[i][j] - mean : 0.f;
      }
    }
  }
  uint64_t q2[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < PACKS; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint64_t e = f32_pair(v[i][j], v[i][j + 1]);
      q2[(j >> 1) & 1] = f32_fma2(e, e, q2[(j >> 1) & 1]);
    }
  float lo, hi;
  f32_unpair(f32_add2(q2[0], q2[1]), lo, hi);
  return rsqrtf(fmaf(row_sum<TPR>(lo + hi, words[1]), inv_dim, eps));
}

// A row's cache lines on their way into L2, one per thread: with a quarter of the warps an SM can hold (a row needs its
// registers), the loads of the next row would otherwise start only when this one is written.
template <typename T, int TPR>
__device__ __forceinline__ void prefetch_row(const T* p, int dim, int t) {
  for (int c = t * (128 / (int)sizeof(T)); c < dim; c += TPR * (128 / (int)sizeof(T)))
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p + c));
}

// POST: the branch is normalised first, so all of it is held at once; without, a pack of it lives only until it is added.
template <typename T, int TPR, int PACKS, bool ALIGNED, bool POST>
__global__ void __launch_bounds__(NORM_THREADS) gated_residual_norm_kernel(const __grid_constant__ NormArgs a) {
  pdl_launch_dependents();
  pdl_wait_prior();
  constexpr int ROWS = NORM_THREADS / TPR;
  __shared__ float s_words[2][5][NORM_THREADS / 32];
  const int t = threadIdx.x % TPR;
  const int sub = threadIdx.x / TPR;
  const int dim = a.dim;
  const bool quantise = a.format >= 0;
  const bool nv = a.format == CDB_NVFP4;
  const int64_t all_rows = quantise ? (a.rows + 127) & ~(int64_t)127 : a.rows;
  const int64_t tiles = quantise ? fp4_panel_tiles(dim, nv) : 0;
  const T* gate = static_cast<const T*>(a.gate);
  const T* weight = static_cast<const T*>(a.weight);
  const T* bias = static_cast<const T*>(a.bias);
  const T* post_weight = static_cast<const T*>(a.post_weight);
  const T* post_bias = static_cast<const T*>(a.post_bias);
  // 16-bit rows without a post norm are loaded a row ahead, into registers: a row's loads are in flight while the one
  // before it is reduced and written.  Elsewhere the registers are short and the next row only moves into L2.
  constexpr bool AHEAD = ALIGNED && sizeof(T) == 2 && !POST && PACKS <= 5;
  uint4 ax[AHEAD ? PACKS : 1], ay[AHEAD ? PACKS : 1];
  auto load_ahead = [&](int64_t row) {
    if constexpr (AHEAD) {
      const int64_t b = row / a.tokens, tok = row - b * a.tokens;
      const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + b * a.x_batch + tok * a.x_row);
      const uint4* yr = reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + b * a.y_batch + tok * a.y_row);
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        const int pk = t + i * TPR;
        const bool in = row < a.rows && pk * 8 < dim;
        ax[i] = in ? __ldcs(xr + pk) : make_uint4(0, 0, 0, 0);
        ay[i] = in && a.y != nullptr ? __ldcs(yr + pk) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  load_ahead((int64_t)blockIdx.x * ROWS + sub);
  int parity = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < all_rows; row += (int64_t)gridDim.x * ROWS, parity ^= 1) {
    if (row >= a.rows) {  // padding of the last panel of block scales (the same for all threads of the row)
      for (int w = t; w < tiles; w += TPR) *reinterpret_cast<uint32_t*>(a.block_scales + fp4_scale_word(row, w, tiles)) = 0u;
      continue;
    }
    const int64_t b = row / a.tokens, tok = row - b * a.tokens;
    const T* xr = static_cast<const T*>(a.x) + b * a.x_batch + tok * a.x_row;
    const int64_t next = row + (int64_t)gridDim.x * ROWS;
    if (!AHEAD && next < a.rows) {
      const int64_t nb = next / a.tokens, nt = next - nb * a.tokens;
      prefetch_row<T, TPR>(static_cast<const T*>(a.x) + nb * a.x_batch + nt * a.x_row, dim, t);
      if (a.y != nullptr) prefetch_row<T, TPR>(static_cast<const T*>(a.y) + nb * a.y_batch + nt * a.y_row, dim, t);
    }
    float v[PACKS][8];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int c = first_column<TPR, ALIGNED>(t, i);
      if constexpr (AHEAD) {
        unpack8<T>(ax[i], v[i]);
      } else if (c < dim) {
        load8<T, ALIGNED, TPR>(xr + c, dim - c, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    }
    if (a.y != nullptr) {
      const T* yr = static_cast<const T*>(a.y) + b * a.y_batch + tok * a.y_row;
      T* xo = static_cast<T*>(a.x_out) + row * dim;
      auto add = [&](int i, int c, const float(&y)[8]) {  // x' of one pack
        float f[8], alpha[8];
        fill8(alpha, a.residual_scale);
        if (gate != nullptr) {
          load8<T, ALIGNED, TPR>(gate + b * a.gate_batch + c, dim - c, f);
          mul8(f, f, alpha);
          fma8(v[i], f, y, v[i]);
        } else {
          fma8(v[i], alpha, y, v[i]);
        }
        store8<T, ALIGNED, TPR>(xo + c, dim - c, v[i]);
      };
      if constexpr (POST) {
        float y[PACKS][8];
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
          const int c = first_column<TPR, ALIGNED>(t, i);
          if (c < dim) {
            load8<T, ALIGNED, TPR>(yr + c, dim - c, y[i]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[i][j] = 0.f;
          }
        }
        const float r = normalise<TPR, PACKS, ALIGNED>(y, a.post, t, dim, a.post_eps, s_words[parity]);
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
          const int c = first_column<TPR, ALIGNED>(t, i);
          if (c < dim) {
            float f[8];
            float g[8];
            fill8(f, r);
            if (post_weight != nullptr) {
              load8<T, ALIGNED, TPR>(post_weight + c, dim - c, g);
              mul8(f, f, g);
            }
            fill8(g, 0.f);
            if (post_bias != nullptr) load8<T, ALIGNED, TPR>(post_bias + c, dim - c, g);
            fma8(y[i], y[i], f, g);
            add(i, c, y[i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
          const int c = first_column<TPR, ALIGNED>(t, i);
          if (c < dim) {
            float y[8];
            if constexpr (AHEAD) unpack8<T>(ay[i], y);
            else load8<T, ALIGNED, TPR>(yr + c, dim - c, y);
            add(i, c, y);
          }
        }
      }
    }
    load_ahead(next);
    if (a.norm == NORM_NONE) continue;
    const float r = normalise<TPR, PACKS, ALIGNED>(v, a.norm, t, dim, a.eps, s_words[parity] + 2);
    uint32_t top[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int c = first_column<TPR, ALIGNED>(t, i);
      top[i] = 0u;
      if (c < dim) {
        float f[8], g[8];
        fill8(f, r);
        if (weight != nullptr) {
          load8<T, ALIGNED, TPR>(weight + c, dim - c, g);
          mul8(f, f, g);
        }
        fill8(g, 0.f);
        if (bias != nullptr) load8<T, ALIGNED, TPR>(bias + c, dim - c, g);
        fma8(v[i], v[i], f, g);
        if (a.scale != nullptr) {
          load8<T, ALIGNED, TPR>(static_cast<const T*>(a.scale) + b * a.scale_batch + c, dim - c, f);
          load8<T, ALIGNED, TPR>(static_cast<const T*>(a.shift) + b * a.shift_batch + c, dim - c, g);
          float one[8];
          fill8(one, 1.f);
          add8(f, f, one);
          fma8(v[i], v[i], f, g);
        }
        if (!quantise) {
          store8<T, ALIGNED, TPR>(static_cast<T*>(a.h_out) + row * dim + c, dim - c, v[i]);
        } else {
          top[i] = round8<T>(v[i]);
        }
      }
    }
    if constexpr (ALIGNED) {
      if (!quantise) continue;
      // From here as in the quantisation kernel, with half an nvfp4 block (a quarter of an mxfp4 block) per thread.
      uint32_t row_top = 0u;
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        if (!nv) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        row_top = max(row_top, top[i]);
      }
      float row_scale = 1.f;
      if (nv) {
        row_scale = fp4_row_scale(__uint_as_float(row_max<TPR>(row_top, s_words[parity][4])));
        if (t == 0) a.row_scales[row] = row_scale;
      }
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        const int p = t + i * TPR, c = p * 8;
        const Fp4Step s = nv ? fp4_block_step<true>(__uint_as_float(top[i]), row_scale) : fp4_block_step<false>(__uint_as_float(top[i]), 1.f);
        const uint32_t codes = nv ? fp4_codes<true>(v[i], s) : fp4_codes<false>(v[i], s);
        if (c < dim) __stcs(reinterpret_cast<uint32_t*>(a.codes + row * (int64_t)(dim >> 1)) + p, codes);
        uint32_t w = c < dim ? s.byte : 0u;
        const int near = nv ? 2 : 4;  // lanes of a block
        w |= __shfl_down_sync(0xffffffffu, w, near) << 8;
        w |= __shfl_down_sync(0xffffffffu, w, 2 * near) << 16;
        const int word = p / (4 * near);
        if (p % (4 * near) == 0 && word < tiles) *reinterpret_cast<uint32_t*>(a.block_scales + fp4_scale_word(row, word, tiles)) = w;
      }
    }
  }
}

template <typename T, int TPR, int PACKS, bool ALIGNED, bool POST>
static int launch_norm(const NormArgs& a, cudaStream_t st) {
  static PerDevice resident;
  const int64_t per_sm = resident.get([]() -> int64_t {
    int n = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, gated_residual_norm_kernel<T, TPR, PACKS, ALIGNED, POST>, NORM_THREADS, 0);
    return n > 0 ? n : 1;
  });
  const int64_t rows = a.format >= 0 ? (a.rows + 127) / 128 * 128 : a.rows;
  const int64_t want = (rows + NORM_THREADS / TPR - 1) / (NORM_THREADS / TPR), cap = per_sm * sm_count();
  CDB_CUDA_CHECK(launch_pdl(gated_residual_norm_kernel<T, TPR, PACKS, ALIGNED, POST>, dim3((unsigned)(want < cap ? want : cap)),
                            dim3(NORM_THREADS), 0, st, a));
  return CDB_OK;
}

// Threads per row: the fewest that hold it in four or five packs of 8 elements, up to eight for the widest rows (64 fp32
// registers).
template <typename T>
static int dispatch_norm(const NormArgs& a, bool aligned, cudaStream_t st) {
  // with 4-bit output the padded block scales need a thread each
  const int packs = a.format >= 0 ? (a.dim + FP4_STEP_COLS - 1) / FP4_STEP_COLS * (FP4_STEP_COLS / 8) : (a.dim + 7) / 8;
#define CDB_N(TPR, PACKS, ALIGNED) \
  if (packs <= TPR * PACKS) return a.post != NORM_NONE ? launch_norm<T, TPR, PACKS, ALIGNED, true>(a, st) : launch_norm<T, TPR, PACKS, ALIGNED, false>(a, st)
  if (aligned) {
    CDB_N(32, 1, true);
    CDB_N(32, 2, true);
    CDB_N(32, 4, true);
    CDB_N(64, 4, true);
    CDB_N(128, 3, true);
    CDB_N(128, 4, true);
    CDB_N(128, 5, true);
    CDB_N(256, 3, true);
    CDB_N(256, 4, true);
    CDB_N(256, 6, true);
    CDB_N(256, 8, true);
  } else {
    CDB_N(32, 4, false);
    CDB_N(256, 2, false);
    CDB_N(256, 8, false);
  }
#undef CDB_N
  return CDB_ERR_UNSUPPORTED;
}

}  // namespace cdb

using namespace cdb;

extern "C" int cdb_gated_residual_norm(const void* args_v, int dtype, void* stream) {
  const cdb_norm_args* in = static_cast<const cdb_norm_args*>(args_v);
  if (!in || dtype < CDB_F32 || dtype > CDB_F16) return CDB_ERR_BAD_ARGUMENT;
  NormArgs a{};
  a.x = in->x; a.y = in->y; a.gate = in->gate; a.post_weight = in->post_weight; a.post_bias = in->post_bias;
  a.weight = in->weight; a.bias = in->bias; a.scale = in->scale; a.shift = in->shift;
  a.x_batch = in->x_batch; a.x_row = in->x_row; a.y_batch = in->y_batch; a.y_row = in->y_row;
  a.gate_batch = in->gate_batch; a.scale_batch = in->scale_batch; a.shift_batch = in->shift_batch;
  a.x_out = in->x_out; a.h_out = in->h_out;
  a.codes = static_cast<uint8_t*>(in->codes);
  a.block_scales = static_cast<uint8_t*>(in->block_scales);
  a.row_scales = in->row_scale;
  a.rows = in->batch * in->tokens;
  a.post = in->post; a.norm = in->norm; a.format = in->format;
  a.residual_scale = in->residual_scale; a.post_eps = in->post_eps; a.eps = in->eps;
  if (in->batch < 0 || in->tokens < 0 || in->dim <= 0 || a.post < 0 || a.post > 2 || a.norm < 0 || a.norm > 2 || a.format < -1 ||
      a.format > CDB_MXFP4)
    return CDB_ERR_BAD_ARGUMENT;
  if (a.rows == 0) return CDB_OK;
  if (in->dim > CDB_NORM_MAX_DIM || in->tokens > INT32_MAX || a.rows > INT32_MAX) return CDB_ERR_TOO_LARGE;
  a.tokens = (int)in->tokens;
  a.dim = (int)in->dim;
  if (!a.x || (a.y != nullptr) != (a.x_out != nullptr) || (!a.y && (a.gate || a.post != NORM_NONE)) || (!a.scale != !a.shift) ||
      (a.norm == NORM_NONE && (a.format >= 0 || a.weight || a.bias || a.scale || !a.y)) ||
      (a.norm != NORM_NONE && a.format < 0 && !a.h_out) ||
      (a.format >= 0 && (!a.codes || !a.block_scales || (a.format == CDB_NVFP4 && !a.row_scales))) ||
      (a.post == NORM_NONE && (a.post_weight || a.post_bias)))
    return CDB_ERR_BAD_ARGUMENT;
  const int per16 = dtype == CDB_F32 ? 4 : 8;  // elements of 16 bytes
  const void* pointers[] = {a.x, a.y, a.gate, a.post_weight, a.post_bias, a.weight, a.bias, a.scale, a.shift, a.x_out, a.h_out};
  bool aligned = a.dim % 8 == 0;
  for (const void* p : pointers) aligned = aligned && aligned16(p);
  const int64_t strides[] = {a.x_batch, a.x_row, a.y_batch, a.y_row, a.gate_batch, a.scale_batch, a.shift_batch};
  for (int64_t s : strides) aligned = aligned && s % per16 == 0;
  if (a.format >= 0 && (!aligned || a.dim % 32 != 0 || !aligned16(a.codes) || !aligned16(a.block_scales))) return CDB_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == CDB_F32) return dispatch_norm<float>(a, aligned, st);
  if (dtype == CDB_BF16) return dispatch_norm<__nv_bfloat16>(a, aligned, st);
  return dispatch_norm<__half>(a, aligned, st);
}
