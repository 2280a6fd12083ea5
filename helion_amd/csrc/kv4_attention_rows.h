// kv4_attention for many rows (a piece of a prompt): 128 rows per workgroup, 32 per wave, over tiles of 64 keys that the
// four waves convert together, once for all rows.  Included by kv4_attention.hip.
//
// Wave w loads the codes of keys 16w .. 16w+15 of a tile (a tile ahead of their use), converts them and puts them into the
// LDS as matrix operands: the 16 bytes of each lane side by side, so that a fragment is written and read without a bank
// conflict and needs no swizzle.  Two buffers: while the waves multiply tile t, the next one is converted into the other.
// Every wave reads all fragments for its own two blocks of 16 rows; scores, statistics and outputs stay in its registers
// and nothing is joined at the end.
//
// What bounds it (2048 new tokens of 32 heads over 10240 keys, head dim 128: bf16 440 us, 0.70 PFLOP/s of the formula's
// products; fp16 496): for 32 keys a wave's MFMAs take 832 cycles (16 for the scores, 32 for the two terms of the weights, 4 for
// their sums, 16 cycles each), its vector instructions about 900, its 16 KB of fragments a quarter of 500 cycles of the LDS;
// two waves per SIMD hide little of that behind each other (an MFMA runs in 49 % of the busy cycles, a vector instruction issues in 53).
// Tried and slower (with one term a weight, 323 us): scores one half tile ahead in the wave (385), equal priorities (338).
//
// A sequence with at most 16 rows (a single token in a mixed batch) is worked on as in ka_few instead.
#define KR_WAVES 4
#define KR_RB 2
#define KR_ROWS (16 * KR_RB * KR_WAVES)
#define KR_KEYS 64
template <int D>
struct KrLds {
  v4i k[2][4][D / 32][64];   // [buffer][block of 16 keys][MFMA][lane]
  v4i v[2][2][D / 16][64];   // [buffer][pair of blocks][MFMA][lane]
  int odd[2][4];             // [buffer][block]: 1 its page does not exist, 2 a value of it is NaN
  uint8_t nan_at[2][4][64];  // the NaN values of each lane, one bit per token (where odd says so)
};

template <int D, int DT, int NQ, int NP>
__global__ __launch_bounds__(KR_WAVES * 64, 2) void hx_kv4_attention_rows(KaArgs a) {
  typedef typename KaT<DT>::T T;
  constexpr int DG = D / 4, KM = D / 32, PB = D / 32, VJ = D / 16, RB = KR_RB;
  constexpr size_t LDS = sizeof(KrLds<D>) > sizeof(KaFewLds<D, KR_WAVES>) ? sizeof(KrLds<D>) : sizeof(KaFewLds<D, KR_WAVES>);
  __shared__ __attribute__((aligned(16))) uint8_t raw[LDS];
  KaSeq q;
  if (!ka_sequence<true>(a, q)) return;
  if (q.rows <= 16) {  // (uniform)
    if (q.block0 == 0) ka_few<D, DT, NQ, NP, 1, KR_WAVES, 2>(a, q, *(KaFewLds<D, KR_WAVES>*)raw);
    return;
  }
  KrLds<D>& lds = *(KrLds<D>*)raw;
  // Two waves share a SIMD, and with equal rights they drift into the same phase and wait for the same pipe: one of them
  // goes first wherever both can (2048 new tokens over 10240 keys 461 -> 441 us, head dim 64 347 -> 328; 8 x 512 over 2048 176 -> 182).
  if (hx_wave_slot() & 1) __builtin_amdgcn_s_setprio(2);
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pm = (1 << a.page_shift) - 1;
  const uint32_t kc_off = r16 * (D / 2) + g * (DG / 2), vc_off = (g * 16 + r16) * (4 * PB);
  const uint32_t ks_off = r16 * PB + (D == 64 ? g >> 1 : g), vs_off = (g * PB + r16 / (512 / D)) * 4;

  for (int base = q.block0 * KR_ROWS; base < q.rows; base += a.blocks * KR_ROWS) {
    const int i_end = (unsigned)(min(base + KR_ROWS, q.rows) - 1) / (unsigned)q.G;
    const int n_keys = a.causal ? max(q.kv_len - q.n_new + i_end + 1, 0) : q.kv_len;  // keys any row of the workgroup sees
    const int tiles = (n_keys + KR_KEYS - 1) / KR_KEYS, last_block = (n_keys - 1) >> 4;
    const int row0 = base + 16 * RB * w;
    const bool active = row0 < q.rows;  // (a wave without rows still converts)
    const int i_first = (unsigned)min(row0, q.rows - 1) / (unsigned)q.G;
    const int see_all = a.causal ? q.kv_len - q.n_new + i_first : q.kv_len - 1;  // last key every row of the wave sees

    v8bf qf[RB][NQ][KM];
    int last[RB];
    ka_queries<D, DT, NQ, RB>(a, q, row0, qf, last);
    v4f o[RB][VJ];
    float mx[RB];
    v4f l[RB];  // sums of the weights as multiplied: rows of ones times them
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      mx[rb] = KA_M0;
      l[rb] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < VJ; ++j) o[rb][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    }

    // ---- this wave's 16 keys of a tile, on their way; every load is in range (see ka_few)
    struct Codes {
      uint32_t k[KM], v[PB], ks, vs;
      int there;
    } x;
    auto page_of = [&](int t) { return ka_scalar(q.table + (min(4 * t + w, last_block) >> (a.page_shift - 4))); };
    auto load = [&](int t, int page) {
      x.there = (unsigned)page < (unsigned)a.pages;
      page = x.there ? page : 0;
      const long at = (((long)page * a.kv_heads + q.h) << a.page_shift) + ((min(4 * t + w, last_block) << 4) & pm);
      const uint8_t *kc = a.kc + at * (D / 2), *vc = a.vc + at * (D / 2);
      if (D == 64) {
        const v2i u = *(const v2i*)(kc + kc_off), y = *(const v2i*)(vc + vc_off);
        x.k[0] = u[0], x.k[1] = u[1], x.v[0] = y[0], x.v[1] = y[1];
      } else {
        const v4i u = *(const v4i*)(kc + kc_off), y = *(const v4i*)(vc + vc_off);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.k[e % KM] = u[e], x.v[e % PB] = y[e];
      }
      x.ks = (a.ks + at * PB)[ks_off];
      x.vs = *(const uint32_t*)(a.vs + at * PB + vs_off);
    };
    auto convert = [&](int t, int buf) {
      const float sc = kv4_scale(x.ks);
#pragma unroll
      for (int m = 0; m < KM; ++m) {
        v4i u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = (int)ka_pair(x.k[m], sc, e);
        lds.k[buf][w][m][lane] = u;
      }
      // Scales behind the last key become small finite ones, those that stand for NaN too (put_nan has them).
      uint32_t vs = x.vs, nan = 0;
      const int left = n_keys - (KR_KEYS * t + 16 * w);
      const bool odd = !x.there || left < 16;  // (uniform)
      const bool byte255 = ((~vs - 0x01010101u) & vs & 0x80808080u) != 0;  // a byte of vs is 255: a byte of ~vs is 0
      if (odd || __builtin_amdgcn_ballot_w64(byte255) != 0) {
        HX_OPAQUE_V(vs);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool there = 4 * g + i < left && x.there, is_nan = ((vs >> (8 * i)) & 255) == 255;
          if (there && is_nan) nan |= 1u << i;
          if (!there || is_nan) vs = (vs & ~(255u << (8 * i))) | (1u << (8 * i));
        }
        if (__builtin_amdgcn_ballot_w64(nan != 0) != 0) {
          lds.nan_at[buf][w][lane] = (uint8_t)nan;
          nan = 2;  // (from here on: of the block)
        }
      }
      if (lane == 0) lds.odd[buf][w] = (x.there ? 0 : 1) | (__builtin_amdgcn_readfirstlane(nan) & 2);
#pragma unroll
      for (int jj = 0; jj < VJ / 2; ++jj) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int byte = i * PB + jj;
          u[i] = ka_pair(x.v[byte / 4], kv4_scale_of(vs, i), byte % 4);
        }
        *((v2i*)&lds.v[buf][w >> 1][2 * jj][lane] + (w & 1)) =
            (v2i){(int)__builtin_amdgcn_perm(u[1], u[0], 0x05040100), (int)__builtin_amdgcn_perm(u[3], u[2], 0x05040100)};
        *((v2i*)&lds.v[buf][w >> 1][2 * jj + 1][lane] + (w & 1)) =
            (v2i){(int)__builtin_amdgcn_perm(u[1], u[0], 0x07060302), (int)__builtin_amdgcn_perm(u[3], u[2], 0x07060302)};
      }
    };

    // ---- the steps of a half tile (32 keys)
    v4f s[RB][2];
    auto scores = [&](int t, int pair, v4f(&to)[RB][2]) {
      const int buf = t & 1;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        v8bf kf[KM];
#pragma unroll
        for (int m = 0; m < KM; ++m) kf[m] = __builtin_bit_cast(v8bf, lds.k[buf][2 * pair + tb][m][lane]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          v4f acc = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
            for (int m = 0; m < KM; ++m) acc = Mfma16<true>::run16(kf[m], qf[rb][n][m], acc);
          to[rb][tb] = acc;
        }
      }
    };
    auto mask = [&](int t, int pair, v4f(&to)[RB][2], int odd) {
      const int key0 = KR_KEYS * t + 32 * pair;
      if (key0 + 31 > see_all || odd != 0) {
        int lane_there = 1;
        HX_OPAQUE_V(lane_there);  // keeps this a branch
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
          const bool there = lane_there && !(lds.odd[t & 1][2 * pair + tb] & 1);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + 16 * tb + 4 * g + e > last[rb] || !there) to[rb][tb][e] = -INFINITY;
        }
      }
    };
    auto vote = [&]() {
      float top[RB];
      bool far = false;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        top[rb] = a.c * hx_max3(hx_max3(s[rb][0][0], s[rb][0][1], s[rb][0][2]), hx_max3(s[rb][0][3], s[rb][1][0], s[rb][1][1]),
                               fmaxf(s[rb][1][2], s[rb][1][3]));
        far |= top[rb] > mx[rb] + KA_STEP;
      }
      if (__builtin_amdgcn_ballot_w64(far) != 0) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          top[rb] = fmaxf(top[rb], __shfl_xor(top[rb], 16));
          top[rb] = fmaxf(top[rb], __shfl_xor(top[rb], 32));
          const float next = top[rb] > mx[rb] + KA_STEP ? top[rb] : mx[rb];
          const float f = __builtin_amdgcn_exp2f(mx[rb] - next);
          mx[rb] = next;
          l[rb] *= f;
#pragma unroll
          for (int j = 0; j < VJ; ++j) o[rb][j] *= f;
        }
      }
    };
    auto weights = [&](v8bf(&pf)[RB][NP]) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][tb][e], a.c, -mx[rb]));
            __bf16 u[NP];
            ka_terms<NP>(p, u);
#pragma unroll
            for (int n = 0; n < NP; ++n) pf[rb][n][4 * tb + e] = u[n];
          }
    };
    v8bf ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (__bf16)1.f;
    auto values = [&](int t, int pair, const v8bf(&pf)[RB][NP]) {
#pragma unroll
      for (int n = NP - 1; n >= 0; --n)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) l[rb] = Mfma16<true>::run16(ones, pf[rb][n], l[rb]);
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        const v8bf vf = __builtin_bit_cast(v8bf, lds.v[t & 1][pair][j][lane]);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) o[rb][j] = Mfma16<true>::run16(vf, pf[rb][n], o[rb][j]);
      }
    };
    auto put_nan = [&](int t, int pair, int odd) {
      if (odd & 2) {  // as in ka_few: the pieces with a NaN, for the queries that see its token
        const int buf = t & 1, key0 = KR_KEYS * t + 32 * pair;
        v8bf bad;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int tb = 2 * pair + (e >> 2);
          bad[e] = (lds.odd[buf][tb] & 2) && ((lds.nan_at[buf][tb][lane] >> (e & 3)) & 1) ? (__bf16)1.f : (__bf16)0.f;
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          v8bf sees;
#pragma unroll
          for (int e = 0; e < 8; ++e) sees[e] = key0 + 16 * (e >> 2) + 4 * g + (e & 3) <= last[rb] ? (__bf16)1.f : (__bf16)0.f;
          const v4f count = Mfma16<true>::run16(bad, sees, (v4f){0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < VJ; ++j)
              if (count[e] > 0.f) o[rb][j][e] = __builtin_nanf("");
        }
      }
    };
    auto odd_of = [&](int t) {
      const v4i f = *(const v4i*)&lds.odd[t & 1][0];
      return __builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]);
    };
    auto half = [&](int t, int pair, int odd) {
      scores(t, pair, s);
      mask(t, pair, s, odd);
      vote();
      v8bf pf[RB][NP];
      weights(pf);
      values(t, pair, pf);
      put_nan(t, pair, odd);
    };

    if (tiles > 0) {
      const int t_last = tiles - 1;
      load(0, page_of(0));
      int next_page = page_of(min(1, t_last));
      convert(0, 0);
      load(min(1, t_last), next_page);
      next_page = page_of(min(2, t_last));
      for (int t = 0; t < tiles; ++t) {
        __syncthreads();  // tile t is in its buffer, and nobody reads the other one any more
        if (t < t_last) {
          convert(t + 1, (t + 1) & 1);
          load(min(t + 2, t_last), next_page);
          next_page = page_of(min(t + 3, t_last));
        }
        if (active) {
          const int odd = odd_of(t);
          half(t, 0, odd);
          half(t, 1, odd);
        }
      }
      __syncthreads();  // the next rows start over with buffer 0
    }

    // ---- element d = (4g + e) * VJ + j of row c is o[j][e] of lane (c, g)
    if (active)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float sum = l[rb][0];
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key gives zeros
        const int row = row0 + 16 * rb + r16;
        if (row < q.rows) {
          const int i = (unsigned)row / (unsigned)q.G, hq = q.h * q.G + row - i * q.G;
          T* dst = (T*)a.out + ((long)(q.start + i) * a.heads + hq) * D;
          typedef T Tv __attribute__((ext_vector_type(VJ)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            Tv v;
#pragma unroll
            for (int j = 0; j < VJ; ++j) v[j] = (T)(o[rb][j][e] * inv);
            *(Tv*)(dst + (4 * g + e) * VJ) = v;
          }
        }
      }
  }
}
