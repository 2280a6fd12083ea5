// Writing tokens into the 4-bit key/value cache and reading them back (format and layout: kv4_format.h).
//
// Both are streams: write reads k and v once and writes D/2 + D/32 bytes per token, head and side; read does the
// opposite.  A lane holds eight consecutive elements of one head of one token: 16 bytes of a 16-bit type, one dword of
// codes; the four lanes of a 32-element block find its maximum with two shuffles.  A wave takes several consecutive
// tokens of one head, so that where their slots are consecutive too (a prompt) the codes of the wave fill whole lines.
#include "hx_common.h"
#include "kv4_format.h"

#include <type_traits>

#define KV4_THREADS 256
#define KV4_BUCKETS 1024

template <int DT>
struct KvT;
template <>
struct KvT<HX_F16> {
  typedef _Float16 T;
};
template <>
struct KvT<HX_BF16> {
  typedef __bf16 T;
};
template <>
struct KvT<HX_F32> {
  typedef float T;
};

struct Kv4Ptrs {  // keys, values
  void* codes[2];
  void* scales[2];
};
struct Kv4Rows {  // the 16- or 32-bit side: [tokens][heads][D], in elements
  const void* p[2];
  long token_stride[2], head_stride[2];
};

// byte offset of this lane's dword of codes (elements 8l .. 8l+7) and of the scale of its block, inside a page of a head
template <int D, bool VALUES>
__device__ __forceinline__ void kv4_place(int in_page, int l, int* code, int* scale) {
  constexpr int PB = D / 32;  // bytes of a piece = scales of a token
  if (VALUES) {
    const int byte = 4 * l;  // (a piece of 2 bytes: the lane's dword is two of them, the second 4 pieces' worth on)
    *code = ((in_page >> 2) * 16 + byte / PB) * 4 * PB + (in_page & 3) * PB + byte % PB;
    *scale = ((in_page >> 2) * PB + l / 4) * 4 + (in_page & 3);
  } else {
    *code = in_page * (D / 2) + 4 * l;
    *scale = in_page * PB + l / 4;
  }
}

// Which of the workgroup's tokens (t0 .. t0+63) are overtaken by a later token with the same slot: bit j of the result.
// Their slots go into a small table; the slots of all later tokens are looked up in it.  The later one wins, whatever
// order the workgroups run in.
template <typename I>
__device__ uint64_t kv4_overtaken(const I* __restrict__ slots, long tokens, long capacity, long t0, int n) {
  __shared__ uint32_t table[2][KV4_BUCKETS];
  __shared__ uint32_t dead[2];
  __shared__ I mine[64];
  for (int i = threadIdx.x; i < 2 * KV4_BUCKETS; i += KV4_THREADS) (&table[0][0])[i] = 0;
  if (threadIdx.x < 2) dead[threadIdx.x] = 0;
  if ((int)threadIdx.x < n) mine[threadIdx.x] = slots[t0 + threadIdx.x];
  __syncthreads();
  if ((int)threadIdx.x < n && mine[threadIdx.x] >= 0 && (long)mine[threadIdx.x] < capacity)
    atomicOr(&table[threadIdx.x >> 5][(uint32_t)mine[threadIdx.x] % KV4_BUCKETS], 1u << (threadIdx.x & 31));
  __syncthreads();
  for (long t = t0 + 1 + threadIdx.x; t < tokens; t += KV4_THREADS) {
    const I s = slots[t];
    const uint32_t b = (uint32_t)s % KV4_BUCKETS;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t m = table[w][b];
      while (m) {
        const int j = __builtin_ctz(m);
        m &= m - 1;
        if (mine[32 * w + j] == s && t0 + 32 * w + j < t) atomicOr(&dead[w], 1u << j);
      }
    }
  }
  __syncthreads();
  return dead[0] | ((uint64_t)dead[1] << 32);
}

template <int D, bool VALUES, typename T>
__device__ __forceinline__ void kv4_put(const T* __restrict__ src, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int in_page,
                                        int l) {
  typedef T Tv __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const Tv raw = *(const Tv*)(src + 8 * l);
  float f[8];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = (float)raw[e];
    top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
  }
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  const uint32_t byte = kv4_scale_byte(top);
  uint32_t c = 0;
  if (byte != 255) {
    const float s = kv4_scale(byte);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
  }
  int at_code, at_scale;
  kv4_place<D, VALUES>(in_page, l, &at_code, &at_scale);
  if (VALUES && D == 64) {  // pieces of two bytes: two of them
    *(uint16_t*)(codes + at_code) = (uint16_t)c;
    *(uint16_t*)(codes + at_code + 8) = (uint16_t)(c >> 16);
  } else {
    *(uint32_t*)(codes + at_code) = c;
  }
  if ((l & 3) == 0) scales[at_scale] = (uint8_t)byte;
}

// Both kernels: grid (groups of `per` tokens, groups of `hb` heads, keys / values); a workgroup takes 256 / (D/8) tokens of
// one head at a time.
template <int DT, int D, typename I>
__global__ __launch_bounds__(KV4_THREADS) void hx_kv4_write_kernel(Kv4Rows rows, Kv4Ptrs cache, const I* __restrict__ slots, long tokens,
                                                                  int heads, int page_shift, long capacity, int per, int hb) {
  typedef typename KvT<DT>::T T;
  constexpr int L = D / 8;              // lanes per row
  constexpr int RPS = KV4_THREADS / L;  // rows at a time
  const long t0 = (long)blockIdx.x * per;
  const int n = (int)min((long)per, tokens - t0);
  const int h0 = blockIdx.y * hb, h1 = min(h0 + hb, heads);
  const uint64_t dead = kv4_overtaken<I>(slots, tokens, capacity, t0, n);
  const int side = blockIdx.z, l = threadIdx.x % L, pm = (1 << page_shift) - 1;
  for (int j = threadIdx.x / L; j < n; j += RPS) {
    const long slot = (long)slots[t0 + j];
    if (slot < 0 || slot >= capacity || ((dead >> j) & 1)) continue;
    const T* src = (const T*)rows.p[side] + (t0 + j) * rows.token_stride[side];
    for (int h = h0; h < h1; ++h) {
      const long at = ((slot >> page_shift) * heads + h) << page_shift;  // tokens in front of this page of this head
      uint8_t* codes = (uint8_t*)cache.codes[side] + at * (D / 2);
      uint8_t* scales = (uint8_t*)cache.scales[side] + at * (D / 32);
      if (side == 0) kv4_put<D, false>(src + h * rows.head_stride[side], codes, scales, (int)(slot & pm), l);
      else kv4_put<D, true>(src + h * rows.head_stride[side], codes, scales, (int)(slot & pm), l);
    }
  }
}

// eight elements of one token of one head as fp32
template <int D, bool VALUES>
__device__ __forceinline__ void kv4_get(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int in_page, int l, float (&f)[8]) {
  int at_code, at_scale;
  kv4_place<D, VALUES>(in_page, l, &at_code, &at_scale);
  uint32_t c;
  if (VALUES && D == 64) c = *(const uint16_t*)(codes + at_code) | ((uint32_t) * (const uint16_t*)(codes + at_code + 8) << 16);
  else c = *(const uint32_t*)(codes + at_code);
  const float s = kv4_scale(scales[at_scale]);
  const v2f p0 = kv4_pair_f32<0>(c, s), p1 = kv4_pair_f32<1>(c, s), p2 = kv4_pair_f32<2>(c, s), p3 = kv4_pair_f32<3>(c, s);
  f[0] = p0[0], f[1] = p0[1], f[2] = p1[0], f[3] = p1[1], f[4] = p2[0], f[5] = p2[1], f[6] = p3[0], f[7] = p3[1];
}

template <int DT, int D, typename I>
__global__ __launch_bounds__(KV4_THREADS) void hx_kv4_read_kernel(Kv4Ptrs cache, Kv4Ptrs out, const I* __restrict__ slots, long tokens,
                                                                 int heads, int page_shift, long capacity, int per, int hb) {
  typedef typename KvT<DT>::T T;
  typedef T Tv __attribute__((ext_vector_type(8)));
  constexpr int L = D / 8;
  constexpr int RPS = KV4_THREADS / L;
  const long t0 = (long)blockIdx.x * per;
  const int n = (int)min((long)per, tokens - t0);
  const int h0 = blockIdx.y * hb, h1 = min(h0 + hb, heads);
  const int side = blockIdx.z, l = threadIdx.x % L, pm = (1 << page_shift) - 1;
  for (int j = threadIdx.x / L; j < n; j += RPS) {
    const long slot = (long)slots[t0 + j];
    const bool there = slot >= 0 && slot < capacity;
    T* dst = (T*)out.codes[side] + (t0 + j) * heads * D;
    for (int h = h0; h < h1; ++h) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (there) {
        const long at = ((slot >> page_shift) * heads + h) << page_shift;
        const uint8_t* codes = (const uint8_t*)cache.codes[side] + at * (D / 2);
        const uint8_t* scales = (const uint8_t*)cache.scales[side] + at * (D / 32);
        if (side == 0) kv4_get<D, false>(codes, scales, (int)(slot & pm), l, f);
        else kv4_get<D, true>(codes, scales, (int)(slot & pm), l, f);
      }
      Tv v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
      *(Tv*)(dst + h * D + 8 * l) = v;
    }
  }
}

// what every entry point of the cache asks of it; 0 or an error
int kv4_check_cache(const char* who, const void* kc, const void* ks, const void* vc, const void* vs, int64_t pages, int64_t page,
                    int64_t heads, int64_t D) {
  if (pages < 0 || heads < 0) {
    hx_set_error("%s: negative size", who);
    return HX_ERR_BAD_ARG;
  }
  if (page < 16 || page > 1024 || (page & (page - 1)) != 0) {
    hx_set_error("%s: pages of a power of two from 16 to 1024 tokens, got %lld", who, (long long)page);
    return HX_ERR_UNSUPPORTED;
  }
  if (D != 64 && D != 128 && D != 256) {
    hx_set_error("%s: head dim 64, 128 or 256, got %lld", who, (long long)D);
    return HX_ERR_UNSUPPORTED;
  }
  if (heads > 65535 || pages > 0x7FFFFFFF) {
    hx_set_error("%s: too many heads or pages", who);
    return HX_ERR_UNSUPPORTED;
  }
  if (pages > 0 && heads > 0 && (!kc || !ks || !vc || !vs)) {
    hx_set_error("%s: null cache pointer", who);
    return HX_ERR_BAD_ARG;
  }
  if ((((uintptr_t)kc | (uintptr_t)ks | (uintptr_t)vc | (uintptr_t)vs) & 15) != 0) {
    hx_set_error("%s: cache pointers must be 16-byte aligned", who);
    return HX_ERR_UNSUPPORTED;
  }
  return 0;
}

static int kv4_shift(int64_t page) { return __builtin_ctzll((unsigned long long)page); }

template <typename F>
static void kv4_pick(int dt, int64_t D, int wide, F&& f) {
  auto by_i = [&](auto dtc, auto dc) {
    if (wide) f(dtc, dc, (int64_t)0);
    else f(dtc, dc, (int32_t)0);
  };
  auto by_d = [&](auto dtc) {
    if (D == 64) by_i(dtc, std::integral_constant<int, 64>{});
    else if (D == 128) by_i(dtc, std::integral_constant<int, 128>{});
    else by_i(dtc, std::integral_constant<int, 256>{});
  };
  if (dt == HX_F16) by_d(std::integral_constant<int, HX_F16>{});
  else if (dt == HX_BF16) by_d(std::integral_constant<int, HX_BF16>{});
  else by_d(std::integral_constant<int, HX_F32>{});
}

static int kv4_check_rows(const char* who, int64_t tokens, int dt, const void* slots, int wide) {
  if (tokens < 0) {
    hx_set_error("%s: negative size", who);
    return HX_ERR_BAD_ARG;
  }
  if (dt != HX_F16 && dt != HX_BF16 && dt != HX_F32) {
    hx_set_error("%s: dtype must be HX_F16, HX_BF16 or HX_F32, got %d", who, dt);
    return HX_ERR_BAD_ARG;
  }
  if (tokens > 0 && !slots) {
    hx_set_error("%s: null pointer", who);
    return HX_ERR_BAD_ARG;
  }
  if (tokens > (1l << 30)) {
    hx_set_error("%s: at most 2^30 tokens, got %lld", who, (long long)tokens);
    return HX_ERR_UNSUPPORTED;
  }
  if ((uintptr_t)slots & (wide ? 7 : 3)) {
    hx_set_error("%s: slots must be aligned to their elements", who);
    return HX_ERR_UNSUPPORTED;
  }
  return 0;
}

// Tokens and heads per workgroup: 64 tokens and all heads keep the look for later tokens of the same slot (every workgroup
// reads the slots behind its own) small next to the data; few tokens are spread over more workgroups instead.
struct Kv4Grid {
  int per, hb;
  unsigned x, y;
};
static Kv4Grid kv4_grid(int64_t tokens, int64_t heads, int64_t D) {
  Kv4Grid g;
  g.per = tokens >= 4096 ? 64 : D == 64 ? 32 : 16;
  g.x = (unsigned)((tokens + g.per - 1) / g.per);
  g.hb = (int)heads;
  while (g.hb > 1 && (long)g.x * ((heads + g.hb - 1) / g.hb) < hx_cu_count()) g.hb = (g.hb + 1) / 2;
  g.y = (unsigned)((heads + g.hb - 1) / g.hb);
  return g;
}

static int kv4_status(const char* who) {
  const hipError_t e = hx_launch_status();
  if (e != hipSuccess) {
    hx_set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}

extern "C" int hx_kv4_write(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes, void* v_scales, const void* slots,
                            int slots_are_int64, int64_t tokens, int64_t heads, int64_t D, int64_t pages, int64_t page,
                            int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                            void* stream) {
  int rc = kv4_check_cache("hx_kv4_write", k_codes, k_scales, v_codes, v_scales, pages, page, heads, D);
  if (rc == 0) rc = kv4_check_rows("hx_kv4_write", tokens, dtype, slots, slots_are_int64);
  if (rc != 0 || tokens == 0 || heads == 0 || pages == 0) return rc;
  if (!k || !v) {
    hx_set_error("hx_kv4_write: null pointer");
    return HX_ERR_BAD_ARG;
  }
  if (((uintptr_t)k | (uintptr_t)v) & (dtype == HX_F32 ? 3 : 1)) {
    hx_set_error("hx_kv4_write: k and v must be aligned to their elements");
    return HX_ERR_UNSUPPORTED;
  }
  const Kv4Grid g = kv4_grid(tokens, heads, D);
  Kv4Rows rows = {{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}};
  Kv4Ptrs cache = {{k_codes, v_codes}, {k_scales, v_scales}};
  kv4_pick(dtype, D, slots_are_int64, [&](auto dtc, auto dc, auto i) {
    typedef decltype(i) I;
    hx_launch(hx_kv4_write_kernel<decltype(dtc)::value, decltype(dc)::value, I>,
              dim3(g.x, g.y, 2), dim3(KV4_THREADS), 0, (hipStream_t)stream, rows, cache, (const I*)slots, (long)tokens, (int)heads,
              kv4_shift(page), (long)(pages * page), g.per, g.hb);
  });
  return kv4_status("hx_kv4_write");
}

extern "C" int hx_kv4_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const void* slots,
                           int slots_are_int64, void* k, void* v, int64_t tokens, int64_t heads, int64_t D, int64_t pages, int64_t page,
                           int dtype, void* stream) {
  int rc = kv4_check_cache("hx_kv4_read", k_codes, k_scales, v_codes, v_scales, pages, page, heads, D);
  if (rc == 0) rc = kv4_check_rows("hx_kv4_read", tokens, dtype, slots, slots_are_int64);
  if (rc != 0 || tokens == 0 || heads == 0) return rc;
  if (!k || !v) {
    hx_set_error("hx_kv4_read: null pointer");
    return HX_ERR_BAD_ARG;
  }
  if (((uintptr_t)k | (uintptr_t)v) & 15) {
    hx_set_error("hx_kv4_read: k and v must be 16-byte aligned");
    return HX_ERR_UNSUPPORTED;
  }
  Kv4Ptrs cache = {{(void*)k_codes, (void*)v_codes}, {(void*)k_scales, (void*)v_scales}}, out = {{k, v}, {nullptr, nullptr}};
  const Kv4Grid g = kv4_grid(tokens, heads, D);
  kv4_pick(dtype, D, slots_are_int64, [&](auto dtc, auto dc, auto i) {
    typedef decltype(i) I;
    hx_launch(hx_kv4_read_kernel<decltype(dtc)::value, decltype(dc)::value, I>, dim3(g.x, g.y, 2), dim3(KV4_THREADS), 0,
              (hipStream_t)stream, cache, out, (const I*)slots, (long)tokens, (int)heads, kv4_shift(page), (long)(pages * page), g.per, g.hb);
  });
  return kv4_status("hx_kv4_read");
}
