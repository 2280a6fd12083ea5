// Writing tokens into the 4-bit key/value cache and reading them back (format and layout: kv4_format.h).
//
// Both are streams, bound by memory: write reads k and v once and writes D/2 + D/32 bytes per token, head and side; read
// does the opposite.  A lane holds eight consecutive elements of one head of one token: 16 bytes of a 16-bit type, one dword of
// codes; the four lanes of a 32-element block find its maximum with two shuffles.  A wave takes several consecutive
// tokens of one head, so that where their slots are consecutive too (a prompt) the codes of the wave fill whole lines.
// Loads of eight heads are on their way at once, and what is read once goes past the caches: 16384 tokens of 8 heads of 128
// written and read back 68 -> 39 us, 172 MB at 4.5 TB/s.
#include "hx_common.h"
#include "kv4_format.h"

#include <type_traits>

#define KV4_THREADS 256
#define KV4_BUCKETS 1024
#define KV4_AHEAD 8          // heads whose loads are on their way before the first is worked on
#define KV4_TURN (1 << 15)   // tokens written by one launch

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

// Which of the workgroup's tokens (t0 .. t0+n-1, n up to 32) are overtaken by a later token with the same slot: bit j of the result.
// Their slots go into a small table; the slots of all later tokens of the launch are looked up in it.  The later one wins, whatever
// order the workgroups run in.
template <typename I>
__device__ uint32_t kv4_overtaken(const I* __restrict__ slots, long tokens, long capacity, long t0, int n) {
  __shared__ uint32_t table[KV4_BUCKETS];
  __shared__ uint32_t dead;
  __shared__ I mine[32];
  for (int i = threadIdx.x; i < KV4_BUCKETS; i += KV4_THREADS) table[i] = 0;
  if (threadIdx.x == 0) dead = 0;
  if ((int)threadIdx.x < n) mine[threadIdx.x] = slots[t0 + threadIdx.x];
  __syncthreads();
  if ((int)threadIdx.x < n && mine[threadIdx.x] >= 0 && (long)mine[threadIdx.x] < capacity)
    atomicOr(&table[(uint32_t)mine[threadIdx.x] % KV4_BUCKETS], 1u << threadIdx.x);
  __syncthreads();
  auto look = [&](I s, long t) {
    uint32_t m = table[(uint32_t)s % KV4_BUCKETS];
    if (m) m &= ~*(volatile uint32_t*)&dead;  // (what another lane has found already need not be found again)
    while (m) {
      const int j = __builtin_ctz(m);
      m &= m - 1;
      if (mine[j] == s && t0 + j < t) atomicOr(&dead, 1u << j);
    }
  };
  constexpr int U = 8;  // slots on their way per lane: the look through a long prompt is a chain of loads otherwise
  long at = t0 + 1 + threadIdx.x;
  for (; at + (U - 1) * KV4_THREADS < tokens; at += U * KV4_THREADS) {
    I s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = slots[at + u * KV4_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) look(s[u], at + u * KV4_THREADS);
  }
  for (; at < tokens; at += KV4_THREADS) look(slots[at], at);
  __syncthreads();
  return dead;
}

template <typename T>
struct Kv4Raw {
  typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <int D, bool VALUES, typename T>
__device__ __forceinline__ void kv4_put(const typename Kv4Raw<T>::V raw, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                        int in_page, int l) {
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
template <int DT, int D, int A, typename I>
__global__ __launch_bounds__(KV4_THREADS) void hx_kv4_write_kernel(Kv4Rows rows, Kv4Ptrs cache, const I* __restrict__ slots, long tokens,
                                                                  int heads, int page_shift, long capacity, int per, int hb) {
  typedef typename KvT<DT>::T T;
  constexpr int L = D / 8;              // lanes per row
  constexpr int RPS = KV4_THREADS / L;  // rows at a time
  const long t0 = (long)blockIdx.x * per;
  const int n = (int)min((long)per, tokens - t0);
  const int h0 = blockIdx.y * hb, h1 = min(h0 + hb, heads);
  const uint32_t dead = kv4_overtaken<I>(slots, tokens, capacity, t0, n);
  const int side = blockIdx.z, l = threadIdx.x % L, pm = (1 << page_shift) - 1;
  for (int j = threadIdx.x / L; j < n; j += RPS) {
    const long slot = (long)slots[t0 + j];
    if (slot < 0 || slot >= capacity || ((dead >> j) & 1)) continue;
    const T* src = (const T*)rows.p[side] + (t0 + j) * rows.token_stride[side] + 8 * l;
    for (int h = h0; h < h1; h += A) {
      typename Kv4Raw<T>::V raw[A];
#pragma unroll
      for (int u = 0; u < A; ++u)
        raw[u] = __builtin_nontemporal_load((const typename Kv4Raw<T>::V*)(src + min(h + u, h1 - 1) * rows.head_stride[side]));
#pragma unroll
      for (int u = 0; u < A; ++u) {
        if (h + u >= h1) break;
        const long at = ((slot >> page_shift) * heads + h + u) << page_shift;  // tokens in front of this page of this head
        uint8_t* codes = (uint8_t*)cache.codes[side] + at * (D / 2);
        uint8_t* scales = (uint8_t*)cache.scales[side] + at * (D / 32);
        if (side == 0) kv4_put<D, false, T>(raw[u], codes, scales, (int)(slot & pm), l);
        else kv4_put<D, true, T>(raw[u], codes, scales, (int)(slot & pm), l);
      }
    }
  }
}

// eight elements of one token of one head: dword of codes and byte of scale
template <int D, bool VALUES>
__device__ __forceinline__ void kv4_get(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int in_page, int l, uint32_t* c,
                                        uint32_t* byte) {
  int at_code, at_scale;
  kv4_place<D, VALUES>(in_page, l, &at_code, &at_scale);
  if (VALUES && D == 64) *c = *(const uint16_t*)(codes + at_code) | ((uint32_t) * (const uint16_t*)(codes + at_code + 8) << 16);
  else *c = *(const uint32_t*)(codes + at_code);
  *byte = scales[at_scale];
}

template <int DT, int D, int A, typename I>
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
    T* dst = (T*)out.codes[side] + (t0 + j) * heads * D + 8 * l;
    for (int h = h0; h < h1; h += A) {
      uint32_t c[A], byte[A];
#pragma unroll
      for (int u = 0; u < A; ++u) {
        c[u] = 0, byte[u] = 127;
        if (!there) continue;
        const long at = ((slot >> page_shift) * heads + min(h + u, h1 - 1)) << page_shift;
        const uint8_t* codes = (const uint8_t*)cache.codes[side] + at * (D / 2);
        const uint8_t* scales = (const uint8_t*)cache.scales[side] + at * (D / 32);
        if (side == 0) kv4_get<D, false>(codes, scales, (int)(slot & pm), l, &c[u], &byte[u]);
        else kv4_get<D, true>(codes, scales, (int)(slot & pm), l, &c[u], &byte[u]);
      }
#pragma unroll
      for (int u = 0; u < A; ++u) {
        if (h + u >= h1) break;
        const float s = kv4_scale(byte[u]);
        const v2f p0 = kv4_pair_f32<0>(c[u], s), p1 = kv4_pair_f32<1>(c[u], s), p2 = kv4_pair_f32<2>(c[u], s), p3 = kv4_pair_f32<3>(c[u], s);
        Tv v;
        v[0] = (T)p0[0], v[1] = (T)p0[1], v[2] = (T)p1[0], v[3] = (T)p1[1], v[4] = (T)p2[0], v[5] = (T)p2[1], v[6] = (T)p3[0], v[7] = (T)p3[1];
        __builtin_nontemporal_store(v, (Tv*)(dst + (long)(h + u) * D));
      }
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
static void kv4_pick(int dt, int64_t D, int hb, int wide, F&& f) {
  auto by_i = [&](auto dtc, auto dc) {
    auto by_a = [&](auto i) {
      if (hb >= 4) f(dtc, dc, std::integral_constant<int, KV4_AHEAD>{}, i);
      else f(dtc, dc, std::integral_constant<int, 1>{}, i);
    };
    if (wide) by_a((int64_t)0);
    else by_a((int32_t)0);
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

// Tokens and heads per workgroup: 32 tokens and all heads keep the look for later tokens of the same slot (every workgroup
// reads the slots behind its own: 3 of the 39 us above) small next to the data, at 64 there are too few workgroups for the
// chip (42 us), at 16 too much looking (41); few tokens are spread over more workgroups, with their heads one by one.
struct Kv4Grid {
  int per, hb;
  unsigned x, y;
};
static Kv4Grid kv4_grid(int64_t tokens, int64_t heads, int64_t D) {
  Kv4Grid g;
  g.per = tokens >= 4096 || D == 64 ? 32 : 16;
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
  // One launch after the other for very many tokens: the look for later ones stays within a launch, and a later launch
  // overwrites an earlier one, so that the work stays proportional to the tokens.
  const int64_t es = dtype == HX_F32 ? 4 : 2;
  Kv4Ptrs cache = {{k_codes, v_codes}, {k_scales, v_scales}};
  for (int64_t first = 0; first < tokens; first += KV4_TURN) {
    const int64_t n = tokens - first < KV4_TURN ? tokens - first : KV4_TURN;
    const Kv4Grid g = kv4_grid(n, heads, D);
    Kv4Rows rows = {{(const char*)k + first * k_token_stride * es, (const char*)v + first * v_token_stride * es},
                    {k_token_stride, v_token_stride},
                    {k_head_stride, v_head_stride}};
    kv4_pick(dtype, D, g.hb, slots_are_int64, [&](auto dtc, auto dc, auto a, auto i) {
      typedef decltype(i) I;
      hx_launch(hx_kv4_write_kernel<decltype(dtc)::value, decltype(dc)::value, decltype(a)::value, I>, dim3(g.x, g.y, 2),
                dim3(KV4_THREADS), 0, (hipStream_t)stream, rows, cache, (const I*)slots + first, (long)n, (int)heads, kv4_shift(page),
                (long)(pages * page), g.per, g.hb);
    });
  }
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
  Kv4Ptrs cache = {{(void*)k_codes, (void*)v_codes}, {(void*)k_scales, (void*)v_scales}};
  const int64_t es = dtype == HX_F32 ? 4 : 2, most = 1l << 20;  // (a launch has room for fewer than 2^32 work-items)
  for (int64_t first = 0; first < tokens; first += most) {
    const int64_t n = tokens - first < most ? tokens - first : most;
    const Kv4Grid g = kv4_grid(n, heads, D);
    const int64_t at = first * heads * D * es;
    Kv4Ptrs out = {{(char*)k + at, (char*)v + at}, {nullptr, nullptr}};
    kv4_pick(dtype, D, g.hb, slots_are_int64, [&](auto dtc, auto dc, auto a, auto i) {
      typedef decltype(i) I;
      hx_launch(hx_kv4_read_kernel<decltype(dtc)::value, decltype(dc)::value, decltype(a)::value, I>, dim3(g.x, g.y, 2), dim3(KV4_THREADS),
                0, (hipStream_t)stream, cache, out, (const I*)slots + first, (long)n, (int)heads, kv4_shift(page), (long)(pages * page), g.per,
                g.hb);
    });
  }
  return kv4_status("hx_kv4_read");
}
