// Row-wise quantisation to 8-bit integers for gfx950, with or without the root-mean-square norm in front of it:
//   hx_rms_norm_int8           h = round_T(x + residual);  y = h * rsqrt(mean(h^2) + eps) * weight
//   hx_int8_quantize_per_token y = x
//   both: scale = max|y| / 127 (1 for a row of zeros),  q = round_to_nearest_even(y * 127 / max|y|)
// so that q * scale ~ y: the (tensor, scale) pairs hx_int8_gemm reads.  h, the residual stream, is rounded to the
// activations' type once and the norm is taken of the rounded values (they are what the next layer adds to).  A row with a NaN
// or an infinity in y gets that as its scale and zeros as its integers.
//
// Precision: the root cancels in y / max|y|, so the integers need only the products h * weight, which fp32 holds exactly for
// 16-bit types (for fp32 they are rounded once), and a quotient that is right next to a middle between two integers (see
// SHORT): a value there falls to the formula's side.  (With plain fp32 quotients one to four of a million integers of a norm
// fell to the other, and 117 of bf16 rows without one, whose quotients are often middles.)  The mean of the squares is summed
// in fp64, where no square of an fp32 number overflows, and the scale is rounded once.
//
// Bound by memory: x (and the residual) are read once, h, q and the scale written once.  A row lives in the registers of
// the lanes that share it, so neither the mean nor the maximum costs a second read; both are reduced together, through the
// wave's shuffles and, where several waves share a row, a few numbers of LDS each.  8192 x 8192 bf16 with a residual:
// 86 us, 470 MB at 5.5 TB/s; one row 4.6 us.
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

// Sum and largest pattern over the TPR lanes that share a row (the whole workgroup, or one wave of four), together: the two
// chains of shuffles run side by side and share a barrier.
template <int TPR>
struct NqLds {
  double sum[TPR / 64];
  unsigned top[2][TPR / 64];
};
template <int TPR, bool SUM>
__device__ __forceinline__ void nq_join(double& sum, unsigned& top, NqLds<TPR>& lds, int turn) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    if (SUM) {
      const uint64_t u = __builtin_bit_cast(uint64_t, sum);
      const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)u, off), hi = (uint32_t)__shfl_xor((int)(uint32_t)(u >> 32), off);
      sum += __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
    }
    top = max(top, (unsigned)__shfl_xor((int)top, off));
  }
  if (TPR == 64) return;
  if ((threadIdx.x & 63) == 0) {
    if (SUM) lds.sum[threadIdx.x >> 6] = sum;
    lds.top[turn][threadIdx.x >> 6] = top;
  }
  __syncthreads();
  top = 0;
#pragma unroll
  for (int i = 0; i < TPR / 64; ++i) top = max(top, lds.top[turn][i]);
  if (SUM) {
    sum = 0.;
#pragma unroll 4  // (sixteen at once would be 32 registers)
    for (int i = 0; i < TPR / 64; ++i) sum += lds.sum[i];
  }
}

// TPR lanes per row, V steps of eight elements per lane: rows of up to 8 * TPR * V elements.
template <int DT, int TPR, int V, bool NORM, bool RES, bool NT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void hx_norm_int8_kernel(
    const typename NqT<DT>::T* __restrict__ x, long x_stride, const typename NqT<DT>::T* __restrict__ res, long res_stride,
    const typename NqT<DT>::T* __restrict__ weight, float eps, double by_width, typename NqT<DT>::T* __restrict__ h_out, signed char* __restrict__ q,
    float* __restrict__ scale, long rows, int width) {
  typedef typename NqT<DT>::T T;
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1;  // rows per workgroup
  __shared__ NqLds<TPR> lds;
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
  double ss = 0.;
  auto times_weight = [&](float unit, int t) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float g[NQ_EPV];
      const int at = (v * TPR + t) * NQ_EPV;
      nq_load<false>(weight + at, width - at, g);
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) y[v][e] = y[v][e] * unit * g[e];
      if (V >= 4) __builtin_amdgcn_sched_barrier(0);  // (the weights of all steps at once would not fit)
    }
  };
  auto largest = [&]() {  // the pattern of |y| as an integer: its order is that of the numbers, with infinity and NaN above them
    unsigned top = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) top = max(top, __float_as_uint(y[v][e]) & 0x7FFFFFFFu);
    return top;
  };
  if (NORM) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) ss = fma((double)y[v][e], (double)y[v][e], ss);
    if (DT != HX_F32) times_weight(1.f, t);
  }
  unsigned top = NORM && DT == HX_F32 ? 0 : largest();
  nq_join<TPR, NORM>(ss, top, lds, 0);
  float unit = 1.f;  // the formula's y is what is in the registers / (unit * rms)
  auto near_one = [&]() {  // a power of two near 1 / rms
    const uint64_t mean = __builtin_bit_cast(uint64_t, fma(ss, by_width, (double)eps));
    const int e2 = 1023 - (int)((mean >> 52) & 0x7FF);
    return __uint_as_float((uint32_t)(min(max(e2 >> 1, -126), 127) + 127) << 23);
  };
  if (NORM && DT == HX_F32) {
    // (one after the other: the second pass below would spill where rows are long, 1024 x 65536 370 us against 316)
    unit = near_one();
    times_weight(unit, t);
    top = largest();
    nq_join<TPR, false>(ss, top, lds, 1);
  } else if (NORM && DT == HX_BF16 && (top >= 0x7F800000u || (top < 0x0D800000u && ss > 0.))) {
    // The largest product has left fp32 or come near its lower end (2^-100): once more, with that power.
    unit = near_one();
    int lane = t;
    HX_OPAQUE_V(lane);  // (addresses of its own: those of the first loads would take their registers all along)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = (v * TPR + lane) * NQ_EPV;
      nq_load<false>((RES ? (const T*)h_out + row * (long)width : x + row * x_stride) + at, width - at, y[v]);
      if (V >= 4) __builtin_amdgcn_sched_barrier(0);
    }
    times_weight(unit, lane);
    top = largest();
    nq_join<TPR, false>(ss, top, lds, 1);
  }
  const float amax = __uint_as_float(top);
  const bool fine = top < 0x7F800000u && top != 0;
  // a maximum near either end of fp32 is moved from there by a power of two, and its row with it
  const float lift = amax < 0x1p-100f ? 0x1p100f : amax > 0x1p100f ? 0x1p-100f : 1.f, most = fine ? amax * lift : 1.f, inv = 1.f / most;
  // The quotient to the nearest integer.  127 times a product of two bf16 numbers, or an fp16 number, has at most 24 bits, and
  // with the remainder of the first guess the fp32 quotient is the correctly rounded one: exact where it is a middle, and no
  // other comes within 2^-24 of itself to one.  127 times a product of fp16 numbers or an fp32 number is rounded, the quotient
  // off by less than 127 * 3 * 2^-24 < 2^-15, and where it lies that near to a middle (one in 2^14) it is worked out in fp64.
  // (A product of fp32 numbers is rounded already.)
  constexpr bool SHORT = DT == HX_BF16 || (DT == HX_F16) != NORM;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = (v * TPR + t) * NQ_EPV;
    signed char c[NQ_EPV];
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < NQ_EPV; ++e) {
      const float p = fine ? y[v][e] * lift * 127.f : 0.f;
      float r = p * inv;
      if (SHORT) r = fmaf(fmaf(-r, most, p), inv, r);
      const float n = rintf(r);
      c[e] = (signed char)(int)n;
      if (!SHORT) off = fmaxf(off, fabsf(r - n));
    }
    if (V >= 4) __builtin_amdgcn_sched_barrier(0);
    if (!SHORT && __builtin_amdgcn_ballot_w64(off > 0.5f - 0x1p-15f) != 0) {
      const double by = 1. / (double)most;
#pragma unroll
      for (int e = 0; e < NQ_EPV; ++e) {
        const double p = fine ? (double)(y[v][e] * lift) * 127. : 0.;
        double r = p * by;
        r = fma(fma(-r, (double)most, p), by, r);
        c[e] = (signed char)(int)rint(r);
        if (V >= 4) __builtin_amdgcn_sched_barrier(0);  // (one at a time: 8192 x 8192 fp16 56 -> 52 us)
      }
    }
    nq_store(q + row * (long)width + at, width - at, c);
  }
  if (t == 0) {  // (last: a chain of roots and quotients that nothing waits for)
    if (NORM) {
      const double rms = sqrt(fma(ss, by_width, (double)eps));
      scale[row] = top == 0 && rms > 0. ? 1.f : (float)((double)amax / ((double)unit * rms * 127.));
    } else {
      scale[row] = top == 0 ? 1.f : (top < 0x7F800000u ? amax / 127.f : amax);
    }
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
                RES ? (const T*)res + at * rs : nullptr, rs, (const T*)w, eps, 1. / width, RES ? (T*)h + at * width : nullptr,
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
