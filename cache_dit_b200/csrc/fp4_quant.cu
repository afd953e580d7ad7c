// 4-bit microscaled quantisation of rows, and back (formats: fp4.cuh).
//
//   cdb_fp4_quant_rows    x [rows, cols] -> codes [rows, cols / 2], block scales (tiled), row scales
//   cdb_fp4_dequant_rows  the values they stand for
//
// Both are one pass over HBM: a thread owns units of 16 columns (32 bytes of a 16-bit type in, 8 bytes of codes out),
// an nvfp4 block; an mxfp4 block is two lanes.  In the nvfp4 kernel a row's threads keep it in registers between the
// row maximum and the conversion.
#include <cstdint>

#include "fp4.cuh"

namespace cdb {

constexpr int FP4_THREADS = 256;

template <typename T>
struct Fp4Unit;  // 16 elements in registers
template <>
struct Fp4Unit<float> {
  float4 v[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldcs(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(int half, float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 t = v[half * 2 + i];
      f[4 * i] = t.x; f[4 * i + 1] = t.y; f[4 * i + 2] = t.z; f[4 * i + 3] = t.w;
    }
  }
  // Largest magnitude.  Compared as integers: an infinity is above every number and a NaN above that.
  __device__ __forceinline__ float top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m = max(m, __float_as_uint(v[i].x) & 0x7fffffffu);
      m = max(m, __float_as_uint(v[i].y) & 0x7fffffffu);
      m = max(m, __float_as_uint(v[i].z) & 0x7fffffffu);
      m = max(m, __float_as_uint(v[i].w) & 0x7fffffffu);
    }
    return __uint_as_float(m);
  }
};
template <typename T>
struct Fp4Unit16 {
  uint4 v[2];
  __device__ __forceinline__ void load(const T* p) {
    v[0] = __ldcs(reinterpret_cast<const uint4*>(p));
    v[1] = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ float to_float(uint32_t bits) {  // bits of one element
    if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16)) return __uint_as_float(bits << 16);
    else return __half2float(__ushort_as_half((unsigned short)bits));
  }
  __device__ __forceinline__ void get(int half, float (&f)[8]) const {
    const uint32_t w[4] = {v[half].x, v[half].y, v[half].z, v[half].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = to_float(w[i] & 0xffffu);
      f[2 * i + 1] = to_float(w[i] >> 16);
    }
  }
  __device__ __forceinline__ float top() const {
    uint32_t m = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m = __vmaxu2(m, __vmaxu2(v[h].x & 0x7fff7fffu, v[h].y & 0x7fff7fffu));
      m = __vmaxu2(m, __vmaxu2(v[h].z & 0x7fff7fffu, v[h].w & 0x7fff7fffu));
    }
    return to_float(max(m & 0xffffu, m >> 16));
  }
};
template <>
struct Fp4Unit<__nv_bfloat16> : Fp4Unit16<__nv_bfloat16> {};
template <>
struct Fp4Unit<__half> : Fp4Unit16<__half> {};

// Maximum of non-negative floats (or NaN) over a warp, as integers.
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// A row is owned by TPR threads, UNITS units each (unit u of the row: thread u % TPR).  Rows beyond `rows` up to the
// next multiple of 128 only get zero scales.
template <typename T, bool NV, int TPR, int UNITS>
__global__ void __launch_bounds__(FP4_THREADS)
    fp4_quant_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ld_x, uint8_t* __restrict__ codes,
                          uint8_t* __restrict__ scales, float* __restrict__ row_scales) {
  pdl_launch_dependents();
  pdl_wait_prior();
  constexpr int ROWS = FP4_THREADS / TPR;  // rows of a CTA at a time
  __shared__ float s_top[2][FP4_THREADS / 32];
  const int t = threadIdx.x % TPR;
  const int sub = threadIdx.x / TPR;
  const int units = cols >> 4;
  const int64_t tiles = fp4_panel_tiles(cols, NV);
  const int64_t all_rows = (rows + 127) & ~(int64_t)127;
  int parity = 0;
  // 16-bit rows are loaded a row ahead: its loads are in flight while the one before it is reduced and written.
  constexpr bool AHEAD = sizeof(T) == 2;
  Fp4Unit<T> ahead[UNITS];
  auto load = [&](int64_t row, Fp4Unit<T>(&u)[UNITS]) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int k = t + i * TPR;
      if (row < rows && k < units) u[i].load(x + row * ld_x + (int64_t)k * 16);
      else u[i].zero();
    }
  };
  if (AHEAD) load((int64_t)blockIdx.x * ROWS + sub, ahead);
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < all_rows; base += (int64_t)gridDim.x * ROWS, parity ^= 1) {
    const int64_t row = base + sub;  // all_rows is a multiple of ROWS
    Fp4Unit<T> u[UNITS];
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < UNITS; ++i) u[i] = ahead[i];
      load(row + (int64_t)gridDim.x * ROWS, ahead);
    } else {
      load(row, u);
    }
    float top[UNITS];
    float row_top = 0.f;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      top[i] = u[i].top();
      if (NV) row_top = __uint_as_float(max(__float_as_uint(row_top), __float_as_uint(top[i])));
      else top[i] = __uint_as_float(max(__float_as_uint(top[i]), __shfl_xor_sync(0xffffffffu, __float_as_uint(top[i]), 1)));
    }
    float row_scale = 1.f;
    if constexpr (NV) {
      row_top = warp_top(row_top);
      if constexpr (TPR > 32) {
        // two slots by parity: a warp that is a row ahead writes the other one, and cannot be two ahead
        if ((threadIdx.x & 31) == 0) s_top[parity][threadIdx.x >> 5] = row_top;
        __syncthreads();
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < TPR / 32; ++w) m = max(m, __float_as_uint(s_top[parity][sub * (TPR / 32) + w]));
        row_top = __uint_as_float(m);
      }
      row_scale = fp4_row_scale(row_top);
      if (t == 0 && row < rows) row_scales[row] = row_scale;
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int k = t + i * TPR;
      const Fp4Step s = fp4_block_step<NV>(top[i], row_scale);
      float f[8];
      uint2 c;
      u[i].get(0, f);
      c.x = fp4_codes<NV>(f, s);
      u[i].get(1, f);
      c.y = fp4_codes<NV>(f, s);
      const bool live = row < rows && k < units;
      if (live) __stcs(reinterpret_cast<uint2*>(codes + row * (int64_t)(cols >> 1)) + k, c);
      // four scales make one word: four neighbouring lanes (nvfp4), or every other one of eight (mxfp4)
      uint32_t w = live ? s.byte : 0u;
      if constexpr (NV) {
        w |= __shfl_down_sync(0xffffffffu, w, 1) << 8;
        w |= __shfl_down_sync(0xffffffffu, w, 2) << 16;
        if ((k & 3) == 0 && (k >> 2) < tiles) *reinterpret_cast<uint32_t*>(scales + fp4_scale_word(row, k >> 2, tiles)) = w;
      } else {
        w |= __shfl_down_sync(0xffffffffu, w, 2) << 8;
        w |= __shfl_down_sync(0xffffffffu, w, 4) << 16;
        if ((k & 7) == 0 && (k >> 3) < tiles) *reinterpret_cast<uint32_t*>(scales + fp4_scale_word(row, k >> 3, tiles)) = w;
      }
    }
  }
}

// 32 bytes at p, in one store where p allows it: two of 16 bytes write every sector in two halves.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8], bool whole) {
  if (whole) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Units of 16 columns, four per thread and step, so that four units' loads are in flight at once.
template <typename T, bool NV>
__global__ void __launch_bounds__(FP4_THREADS)
    fp4_dequant_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                            const float* __restrict__ row_scales, int64_t rows, int cols, T* __restrict__ out) {
  pdl_launch_dependents();
  pdl_wait_prior();
  constexpr int AT_ONCE = 4;
  const int units = cols >> 4;
  const int64_t tiles = fp4_panel_tiles(cols, NV);
  const int64_t total = rows * units;
  const int64_t stride = (int64_t)gridDim.x * FP4_THREADS;
  const bool whole = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
  for (int64_t i0 = (int64_t)blockIdx.x * FP4_THREADS + threadIdx.x; i0 < total; i0 += AT_ONCE * stride) {
    uint2 c[AT_ONCE];
    uint32_t byte[AT_ONCE];
    float row_scale[AT_ONCE];
#pragma unroll
    for (int n = 0; n < AT_ONCE; ++n) {
      const int64_t i = i0 + n * stride;
      if (i < total) {
        const int64_t row = total <= UINT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)units) : i / units;
        const int k = (int)(i - row * units);
        const int b = NV ? k : k >> 1;
        c[n] = __ldcs(reinterpret_cast<const uint2*>(codes) + i);
        byte[n] = __ldg(scales + fp4_scale_word(row, b >> 2, tiles) + (b & 3));
        row_scale[n] = NV ? __ldg(row_scales + row) : 1.f;
      }
    }
#pragma unroll
    for (int n = 0; n < AT_ONCE; ++n) {
      const int64_t i = i0 + n * stride;
      if (i >= total) break;
      float step = fp4_scale_value<NV>(byte[n]);
      if (NV) step *= row_scale[n];
      T* dst = out + i * 16;
      uint32_t w[16];  // 16 numbers of T
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[4];
        e2m1x8_to_half2(h ? c[n].y : c[n].x, p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float2 v = __half22float2(*reinterpret_cast<__half2*>(&p[j]));
          v.x *= step;
          v.y *= step;
          if constexpr (sizeof(T) == 4) {
            w[h * 8 + 2 * j] = __float_as_uint(v.x);
            w[h * 8 + 2 * j + 1] = __float_as_uint(v.y);
          } else if constexpr (__is_same(T, __nv_bfloat16)) {
            const __nv_bfloat162 q = __floats2bfloat162_rn(v.x, v.y);
            w[h * 4 + j] = *reinterpret_cast<const uint32_t*>(&q);
          } else {
            const __half2 q = __floats2half2_rn(v.x, v.y);
            w[h * 4 + j] = *reinterpret_cast<const uint32_t*>(&q);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < (int)sizeof(T) / 2; ++x) {
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = w[x * 8 + j];
        store32(reinterpret_cast<uint8_t*>(dst) + x * 32, u, whole);
      }
    }
  }
}

template <typename T, bool NV, int TPR, int UNITS>
static int launch_quant(const void* x, int64_t rows, int cols, int64_t ld_x, void* codes, void* scales, float* row_scales,
                        cudaStream_t st) {
  static PerDevice resident;
  const int64_t per_sm = resident.get([]() -> int64_t {
    int n = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fp4_quant_rows_kernel<T, NV, TPR, UNITS>, FP4_THREADS, 0);
    return n > 0 ? n : 1;
  });
  const int64_t all_rows = (rows + 127) / 128 * 128;
  const int64_t want = all_rows / (FP4_THREADS / TPR), cap = per_sm * sm_count();
  CDB_CUDA_CHECK(launch_pdl(fp4_quant_rows_kernel<T, NV, TPR, UNITS>, dim3((unsigned)(want < cap ? want : cap)),
                            dim3(FP4_THREADS), 0, st, static_cast<const T*>(x), rows, cols, ld_x,
                            static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), row_scales));
  return CDB_OK;
}

// Threads per row: the fewest that hold the row's padded units, three to five per thread, so that rows of one warp need no
// block barrier and a CTA has several rows in flight.  All padded units need a thread: it writes their zero scales.
template <typename T, bool NV>
static int dispatch_quant(const void* x, int64_t rows, int cols, int64_t ld_x, void* codes, void* scales,
                          float* row_scales, cudaStream_t st) {
  const int units = (cols + FP4_STEP_COLS - 1) / FP4_STEP_COLS * (FP4_STEP_COLS / 16);
#define CDB_Q(TPR, UNITS) \
  if (units <= TPR * UNITS) return launch_quant<T, NV, TPR, UNITS>(x, rows, cols, ld_x, codes, scales, row_scales, st)
  CDB_Q(32, 1);
  CDB_Q(32, 2);
  CDB_Q(32, 4);
  CDB_Q(64, 3);
  CDB_Q(64, 4);
  CDB_Q(64, 5);
  CDB_Q(128, 3);
  CDB_Q(128, 4);
  CDB_Q(256, 4);
#undef CDB_Q
  return CDB_ERR_UNSUPPORTED;
}

}  // namespace cdb

using namespace cdb;

extern "C" size_t cdb_fp4_block_scale_bytes(int64_t rows, int64_t cols, int format) {
  if (rows <= 0 || cols <= 0 || (format != CDB_NVFP4 && format != CDB_MXFP4)) return 0;
  return (size_t)((rows + 127) / 128) * (size_t)fp4_panel_tiles(cols, format == CDB_NVFP4) * 512;
}

static int check_fp4(const void* codes, const void* scales, const float* row_scale, int64_t rows, int64_t cols, int format) {
  if ((format != CDB_NVFP4 && format != CDB_MXFP4) || rows < 0 || cols <= 0) return CDB_ERR_BAD_ARGUMENT;
  if (rows > 0 && (!codes || !scales || (format == CDB_NVFP4 && !row_scale))) return CDB_ERR_BAD_ARGUMENT;
  if (cols % 32 != 0 || cols > FP4_MAX_COLS || rows > INT32_MAX || !aligned16(codes) || !aligned16(scales)) return CDB_ERR_UNSUPPORTED;
  return CDB_OK;
}

extern "C" int cdb_fp4_quant_rows(const void* x, int64_t rows, int64_t cols, int64_t ld_x, int dtype, int format,
                                  void* codes, void* block_scales, float* row_scale, void* stream) {
  const int rc = check_fp4(codes, block_scales, row_scale, rows, cols, format);
  if (rc != CDB_OK) return rc;
  if (rows == 0) return CDB_OK;
  if (!x || ld_x < cols || dtype < CDB_F32 || dtype > CDB_F16) return CDB_ERR_BAD_ARGUMENT;
  if (!aligned16(x) || ld_x % (dtype == CDB_F32 ? 4 : 8) != 0) return CDB_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CDB_D(T)                                                                                                    \
  return format == CDB_NVFP4 ? dispatch_quant<T, true>(x, rows, (int)cols, ld_x, codes, block_scales, row_scale, st) \
                             : dispatch_quant<T, false>(x, rows, (int)cols, ld_x, codes, block_scales, row_scale, st)
  if (dtype == CDB_F32) { CDB_D(float); }
  if (dtype == CDB_BF16) { CDB_D(__nv_bfloat16); }
  CDB_D(__half);
#undef CDB_D
}

extern "C" int cdb_fp4_dequant_rows(const void* codes, const void* block_scales, const float* row_scale, int64_t rows,
                                    int64_t cols, int format, void* out, int dtype, void* stream) {
  const int rc = check_fp4(codes, block_scales, row_scale, rows, cols, format);
  if (rc != CDB_OK) return rc;
  if (rows == 0) return CDB_OK;
  if (!out || dtype < CDB_F32 || dtype > CDB_F16) return CDB_ERR_BAD_ARGUMENT;
  if (!aligned16(out)) return CDB_ERR_UNSUPPORTED;
  const int64_t want = (rows * (cols >> 4) + FP4_THREADS - 1) / FP4_THREADS, cap = (int64_t)sm_count() * 8;
  const dim3 grid((unsigned)(want < cap ? want : cap));
  const uint8_t* cp = static_cast<const uint8_t*>(codes);
  const uint8_t* sp = static_cast<const uint8_t*>(block_scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CDB_D(T)                                                                                                        \
  CDB_CUDA_CHECK(format == CDB_NVFP4                                                                                    \
                     ? launch_pdl(fp4_dequant_rows_kernel<T, true>, grid, dim3(FP4_THREADS), 0, st, cp, sp, row_scale, \
                                  rows, (int)cols, static_cast<T*>(out))                                               \
                     : launch_pdl(fp4_dequant_rows_kernel<T, false>, grid, dim3(FP4_THREADS), 0, st, cp, sp, row_scale, \
                                  rows, (int)cols, static_cast<T*>(out)))
  if (dtype == CDB_F32) CDB_D(float);
  else if (dtype == CDB_BF16) CDB_D(__nv_bfloat16);
  else CDB_D(__half);
#undef CDB_D
  return CDB_OK;
}
