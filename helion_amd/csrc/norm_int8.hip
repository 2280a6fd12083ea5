// Row-wise quantisation to 8-bit integers for gfx950, with or without the root-mean-square norm in front of it:
//   hx_rms_norm_int8           h = round_T(x + residual);  y = h * rsqrt(mean(h^2) + eps) * weight
//   hx_int8_quantize_per_token y = x
//   both: scale = max|y| / 127 (1 for a row of zeros),  q = round_to_nearest_even(y * 127 / max|y|)
// so that q * scale ~ y: the (tensor, scale) pairs hx_int8_gemm reads.  h, the residual stream, is rounded to the
// activations' type once and the norm is taken of the rounded values (they are what the next layer adds to); everything
// from there to q stays in fp32.  A row with a NaN or an infinity in y gets that as its scale and zeros as its integers.
//
// Bound by memory: x (and the residual) are read once, h, q and the scale written once.  A row lives in the registers of
// the lanes that share it, so neither the mean nor the maximum costs a second read; the two reductions go through the
// wave's shuffles and, where several waves share a row, four or sixteen floats of LDS.  8192 x 8192 bf16 with a residual:
// 89 us, 470 MB at 5.3 TB/s; one row 4.1 us.
#include "hx_common.h"

#include <type_traits>

#define NQ_EPV 8  // elements per lane and step: 16 bytes of a 16-bit type

template <int DT>
struct NqT;
template <>
struct NqT<HX_F16> {
  typedef _Float16 T;
};
template <>
struct NqT<HX_BF16> {
  typedef __bf16 T;
};
template <>
struct NqT<HX_F32> {
  typedef float T;
};

// Eight elements at any alignment of the element itself (global loads and stores of 16 bytes need no more on this chip),
// the last ones of a row one by one.
template <bool NT, typename T>
__device__ __forceinline__ void nq_load(const T* __restrict__ p, int left, float (&f)[NQ_EPV]) {
  typedef T Tv __attribute__((ext_vector_type(NQ_EPV), aligned(sizeof(T))));
  if (left >= NQ_EPV) {
    const Tv v = NT ? __builtin_nontemporal_load((const Tv*)p) : *(const Tv*)p;
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) f[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) f[e] = e < left ? (float)p[e] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void nq_store(T* __restrict__ p, int left, const T (&f)[NQ_EPV]) {
  typedef T Tv __attribute__((ext_vector_type(NQ_EPV), aligned(sizeof(T))));
  if (left >= NQ_EPV) {
    Tv v;
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) v[e] = f[e];
    *(Tv*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e)
      if (e < left) p[e] = f[e];
  }
}

// Sum / largest pattern over the TPR lanes that share a row (the whole workgroup, or one wave of four)
template <int TPR>
__device__ __forceinline__ float nq_sum(float v, float* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  if (TPR == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) s += red[i];
  return s;
}
template <int TPR>
__device__ __forceinline__ unsigned nq_max(unsigned v, unsigned* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, off));
  if (TPR == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned s = 0;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) s = max(s, red[i]);
  return s;
}

// TPR lanes per row, V steps of eight elements per lane: rows of up to 8 * TPR * V elements.
template <int DT, int TPR, int V, bool NORM, bool RES, bool NT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void hx_norm_int8_kernel(
    const typename NqT<DT>::T* __restrict__ x, long x_stride, const typename NqT<DT>::T* __restrict__ res, long res_stride,
    const typename NqT<DT>::T* __restrict__ weight, float eps, typename NqT<DT>::T* __restrict__ h_out, signed char* __restrict__ q,
    float* __restrict__ scale, long rows, int width) {
  typedef typename NqT<DT>::T T;
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1;  // rows per workgroup
  __shared__ float red_sum[TPR / 64];
  __shared__ unsigned red_max[TPR / 64];
  const long row = (long)blockIdx.x * RPW + (RPW > 1 ? threadIdx.x / TPR : 0);
  const int t = RPW > 1 ? threadIdx.x % TPR : threadIdx.x;
  if (row >= rows) return;  // (a whole wave leaves: with RPW > 1 a wave is a row and nothing below is shared)

  float y[V][NQ_EPV];
#pragma unroll
  for (int v = 0; v < V; ++v) nq_load<NT>(x + row * x_stride + (v * TPR + t) * NQ_EPV, width - (v * TPR + t) * NQ_EPV, y[v]);
  if (RES) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float r[NQ_EPV];
      T h[NQ_EPV];
      const int at = (v * TPR + t) * NQ_EPV;
      nq_load<NT>(res + row * res_stride + at, width - at, r);
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) {
        h[e] = (T)(y[v][e] + r[e]);
        y[v][e] = (float)h[e];
      }
      nq_store(h_out + row * (long)width + at, width - at, h);
    }
  }
  if (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) ss = fmaf(y[v][e], y[v][e], ss);
    const float rms = sqrtf(nq_sum<TPR>(ss, red_sum) / (float)width + eps);
    const float rstd = 1.f / rms;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float g[NQ_EPV];
      const int at = (v * TPR + t) * NQ_EPV;
      nq_load<false>(weight + at, width - at, g);
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) y[v][e] = y[v][e] * rstd * g[e];
    }
  }
  // the pattern of |y| as an integer: its order is that of the numbers, with infinity and NaN above them
  unsigned top = 0;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) top = max(top, __float_as_uint(y[v][e]) & 0x7FFFFFFFu);
  top = nq_max<TPR>(top, red_max);
  const float amax = __uint_as_float(top);
  const bool fine = top < 0x7F800000u && top != 0;
  // a maximum so small that 127 / amax overflows is lifted by a power of two, and its row with it
  const float lift = amax < 0x1p-100f ? 0x1p100f : 1.f;
  const float inv = fine ? 127.f / (amax * lift) : 0.f;
  if (t == 0) scale[row] = top == 0 ? 1.f : (top < 0x7F800000u ? amax / 127.f : amax);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = (v * TPR + t) * NQ_EPV;
    signed char c[NQ_EPV];
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) c[e] = fine ? (signed char)(int)rintf(y[v][e] * lift * inv) : (signed char)0;
    nq_store(q + row * (long)width + at, width - at, c);
  }
}

template <int DT, bool NORM, bool RES, bool NT>
static void nq_launch(const void* x, long xs, const void* res, long rs, const void* w, float eps, void* h, void* q, float* scale,
                      long rows, int width, hipStream_t s) {
  typedef typename NqT<DT>::T T;
  // rows of thousands of elements by sixteen waves instead of four while there are not enough of them to fill the chip
  // (1 x 8192: 5.6 -> 4.1 us)
  const bool few = rows <= 2 * hx_cu_count();
  auto go = [&](auto kernel, int tpr) {
    const int rpw = tpr < 256 ? 256 / tpr : 1;
    const long most = (1l << 31) / tpr;  // (a launch has room for fewer than 2^32 work-items)
    for (long at = 0; at < rows; at += most) {
      const long n = rows - at < most ? rows - at : most;
      hx_launch(kernel, dim3((unsigned)((n + rpw - 1) / rpw)), dim3(tpr < 256 ? 256 : tpr), 0, s, (const T*)x + at * xs, xs,
                RES ? (const T*)res + at * rs : nullptr, rs, (const T*)w, eps, RES ? (T*)h + at * width : nullptr,
                (signed char*)q + at * width, scale + at, n, width);
    }
  };
  if (width <= 512) go(hx_norm_int8_kernel<DT, 64, 1, NORM, RES, NT>, 64);
  else if (width <= 1024) go(hx_norm_int8_kernel<DT, 64, 2, NORM, RES, NT>, 64);
  else if (width <= 2048) go(hx_norm_int8_kernel<DT, 256, 1, NORM, RES, NT>, 256);
  else if (width <= 4096) go(hx_norm_int8_kernel<DT, 256, 2, NORM, RES, NT>, 256);
  else if (width <= 8192 && few) go(hx_norm_int8_kernel<DT, 1024, 1, NORM, RES, NT>, 1024);
  else if (width <= 8192) go(hx_norm_int8_kernel<DT, 256, 4, NORM, RES, NT>, 256);
  else if (width <= 16384) go(hx_norm_int8_kernel<DT, 1024, 2, NORM, RES, NT>, 1024);
  else if (width <= 32768) go(hx_norm_int8_kernel<DT, 1024, 4, NORM, RES, NT>, 1024);
  else go(hx_norm_int8_kernel<DT, 1024, 8, NORM, RES, NT>, 1024);
}

static int nq_run(const char* who, bool norm, const void* x, int64_t xs, const void* res, int64_t rs, const void* w, float eps, void* h,
                  void* q, float* scale, int64_t rows, int64_t width, int dt, void* stream) {
  if (rows < 0 || width < 0) {
    hx_set_error("%s: negative size", who);
    return HX_ERR_BAD_ARG;
  }
  if (dt != HX_F16 && dt != HX_BF16 && dt != HX_F32) {
    hx_set_error("%s: dtype must be HX_F16, HX_BF16 or HX_F32, got %d", who, dt);
    return HX_ERR_BAD_ARG;
  }
  if (rows == 0) return 0;
  if (width == 0 || width > 65536) {
    hx_set_error("%s: rows of 1 to 65536 elements, got %lld", who, (long long)width);
    return HX_ERR_UNSUPPORTED;
  }
  if (rows > 0x7FFFFFFF) {
    hx_set_error("%s: at most 2^31 - 1 rows, got %lld", who, (long long)rows);
    return HX_ERR_UNSUPPORTED;
  }
  if (!x || !q || !scale || (norm && !w) || (res && !h)) {
    hx_set_error("%s: null pointer", who);
    return HX_ERR_BAD_ARG;
  }
  if ((rows > 1 && xs < width) || (res && rows > 1 && rs < width)) {
    hx_set_error("%s: row stride smaller than the row", who);
    return HX_ERR_BAD_ARG;
  }
  const uintptr_t es = dt == HX_F32 ? 4 : 2;
  if ((((uintptr_t)x | (uintptr_t)res | (uintptr_t)w | (uintptr_t)h) & (es - 1)) != 0 || ((uintptr_t)scale & 3) != 0) {
    hx_set_error("%s: pointers must be aligned to their elements", who);
    return HX_ERR_UNSUPPORTED;
  }
  hipStream_t s = (hipStream_t)stream;
  // x and the residual are read once: past the caches, which what is written then keeps for its reader (8192 x 8192 with a
  // residual, the norm and a product of its integers 267 -> 244 us; 8192 x 4096 126 -> 122), but not where rows begin inside
  // the 16 bytes of a lane, whose lines two lanes' loads share (1968 x 2674: 28.3, past the caches 30.5).
  const bool nt = (((uintptr_t)x | (uintptr_t)res | (uintptr_t)(xs * es) | (uintptr_t)(res ? rs * es : 0)) & 15) == 0;
  auto pick_nt = [&](auto dtc, auto ntc) {
    constexpr int DT = decltype(dtc)::value;
    constexpr bool NT = decltype(ntc)::value;
    if (!norm) nq_launch<DT, false, false, NT>(x, xs, res, rs, w, eps, h, q, scale, rows, (int)width, s);
    else if (!res) nq_launch<DT, true, false, NT>(x, xs, res, rs, w, eps, h, q, scale, rows, (int)width, s);
    else nq_launch<DT, true, true, NT>(x, xs, res, rs, w, eps, h, q, scale, rows, (int)width, s);
  };
  auto pick = [&](auto dtc) {
    if (nt) pick_nt(dtc, std::true_type{});
    else pick_nt(dtc, std::false_type{});
  };
  if (dt == HX_F16) pick(std::integral_constant<int, HX_F16>{});
  else if (dt == HX_BF16) pick(std::integral_constant<int, HX_BF16>{});
  else pick(std::integral_constant<int, HX_F32>{});
  const hipError_t e = hx_launch_status();
  if (e != hipSuccess) {
    hx_set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}

extern "C" int hx_rms_norm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                                float eps, void* h_out, void* q, float* scale, int64_t rows, int64_t width, int dtype, void* stream) {
  return nq_run("hx_rms_norm_int8", true, x, x_stride, residual, residual_stride, weight, eps, h_out, q, scale, rows, width, dtype, stream);
}

extern "C" int hx_int8_quantize_per_token(const void* x, int64_t x_stride, void* q, float* scale, int64_t rows, int64_t width, int dtype,
                                          void* stream) {
  return nq_run("hx_int8_quantize_per_token", false, x, x_stride, nullptr, 0, nullptr, 0.f, nullptr, q, scale, rows, width, dtype, stream);
}
