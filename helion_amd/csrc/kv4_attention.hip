// Attention over the 4-bit key/value cache (format and layout: kv4_format.h), for new tokens of many sequences at once:
//   out[t, hq] = sum_j p_j v[j, hq / G] / sum_j p_j,   p_j = 2^(c (q[t, hq] . k[j, hq / G]) - m),  c = scale * log2(e)
// over the keys j the token may see, in one pass with a running reference point m and sum.  G = query heads per key/value
// head; the keys of sequence b are the first seq_lens[b] slots of its row of the page table.
//
// Precision: an e2m1 value times a power of two is a bf16 number, so keys and values enter the matrix instructions
// exactly.  The other operand of each product is a sum of bf16 terms: one for a bf16 query, two for fp16 (11 bits fit in
// 16), three for fp32; p as two terms (2^-17 of it is lost) or three for fp32, in every kernel, so that a row's precision
// does not depend on the batch around it.  (One term for a bf16 result is faster, 322 instead of 438 us for 2048 new tokens
// over 10240 keys, but then the weights' rounding adds to the result's: 1.4 times its error.)  Products are summed in fp32,
// as are the statistics.
//
// Work: a workgroup takes RB blocks of 16 rows (a row = a new token of one query head) of one sequence and one key/value
// head, so that all G heads share what is read and converted; its waves take key tiles of 32 tokens in turn, each with a
// statistic and an output of its own, joined through the LDS at the end.  Where rows are few the keys are split over
// several workgroups, whose results (fp32, unnormalised) a second kernel joins.
//
// A tile never passes through the LDS: lane (r = lane % 16, g = lane / 16) loads D/4 consecutive elements of key 16 tb + r
// (tb = 0, 1) and the pieces r of the four values 16 tb + 4g .. +3.  S^T = K Q^T (16x16x32, rows = keys) leaves lane (c, g)
// with the scores of query c for the keys 16 tb + 4g + 0..3: exactly the keys whose values the lane holds, so the scores,
// turned into p, are the second operand of O^T += V^T P^T without a move between lanes.  MFMA j of that product has
// element r * D/16 + j of the values as its row r: nibble j of the piece.
#include "hx_common.h"
#include "kv4_format.h"

#include <type_traits>

#define KA_M0 (-3e38f)  // the reference point of a row that has seen no key
#define KA_PIECE 1024  // keys of a split at least
#define KA_GRID (1l << 22)  // workgroups of a launch at most (2^32 work-items are too many for one)
#define KA_STEP 8.f     // it moves only when a score lies 2^8 above it: p stays below 256, and few tiles rescale O

int kv4_check_cache(const char* who, const void* kc, const void* ks, const void* vc, const void* vs, int64_t pages, int64_t page,
                    int64_t heads, int64_t D);

struct KaArgs {
  const void* q;
  long q_token_stride, q_head_stride;  // elements
  void* out;                           // [tokens][heads][D]
  const uint8_t *kc, *ks, *vc, *vs;
  const int* table;
  long table_stride;
  const int *seq_lens, *query_start;
  float* part_o;   // [tokens * heads][splits][D]
  float* part_ml;  // [tokens * heads][splits][2]
  float c;         // |softmax scale| * log2(e); a negative scale turns the queries around instead
  int tokens, batch, heads, kv_heads, pages, page_shift, table_width, causal, splits, blocks, negate, last_first, longest_first, len_shift;
};

template <int DT>
struct KaT;
template <>
struct KaT<HX_F16> {
  typedef _Float16 T;
};
template <>
struct KaT<HX_BF16> {
  typedef __bf16 T;
};
template <>
struct KaT<HX_F32> {
  typedef float T;
};

// a wave-uniform integer that no kernel writes: through the scalar cache
__device__ __forceinline__ int ka_scalar(const int* p) { return *HX_CONSTANT(int, p); }

// byte `sel` (a constant once the loops are unrolled) of `codes` as two bf16 in one register
__device__ __forceinline__ uint32_t ka_pair(uint32_t codes, float scale, int sel) {
  v2bf p;
  switch (sel) {
    case 0: p = kv4_pair_bf16<0>(codes, scale); break;
    case 1: p = kv4_pair_bf16<1>(codes, scale); break;
    case 2: p = kv4_pair_bf16<2>(codes, scale); break;
    default: p = kv4_pair_bf16<3>(codes, scale); break;
  }
  return __builtin_bit_cast(uint32_t, p);
}

// codes that the launch reads once (one block of rows) do not displace what is reused
template <bool NT, typename V>
__device__ __forceinline__ V ka_codes(const V* p) {
  return NT ? __builtin_nontemporal_load(p) : *p;
}

// f = t[0] + t[1] + .. + t[N-1] with bf16 terms, each the rounding of what the ones before it leave
template <int N>
__device__ __forceinline__ void ka_terms(float f, __bf16 (&t)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    t[n] = (__bf16)f;
    f -= (float)t[n];
  }
}

// One sequence and key/value head of a launch
struct KaSeq {
  int b, h, split, block0;
  int G, start, n_new, rows, kv_len;
  const int* table;
};
// The sequence that runs at place `at` of the batch's order: those with more keys first, so that what runs last is short.
// Sequences i * n + g form group g of n groups of up to 64; the groups are taken in turn, each in the order of its lengths
// (in 256 steps of the table's width, equal ones by their number): a lane per sequence, and the length's bits from the top
// down tell in which half of those left the wanted place lies.  64 sequences of up to 2048 keys, 32 heads: 50.7 -> 40.9 us;
// 24 of up to 4000 with 1 to 200 new tokens: 113 -> 103 (both in a graph).
__device__ __forceinline__ int ka_longest_first(const KaArgs& a, int at) {
  const int n = (a.batch + 63) >> 6, g = n == 1 ? 0 : at % n, lane = threadIdx.x & 63;
  int k = n == 1 ? at : at / n;
  const int i = lane * n + g;
  const long most = (long)a.table_width << a.page_shift;
  const int len = (int)min((long)max(i < a.batch ? a.seq_lens[i] : 0, 0), most) >> a.len_shift;
  uint64_t left = __builtin_amdgcn_ballot_w64(i < a.batch);
#pragma unroll
  for (int bit = 7; bit >= 0; --bit) {
    const uint64_t longer = __builtin_amdgcn_ballot_w64((len >> bit) & 1) & left;
    const int c = __builtin_popcountll(longer);
    left = k < c ? longer : left & ~longer;
    k -= k < c ? 0 : c;
  }
  const bool me = ((left >> lane) & 1) && __builtin_popcountll(left & ((1ull << lane) - 1)) == k;
  return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__builtin_amdgcn_ballot_w64(me)) * n + g);
}
template <bool MANY>
__device__ __forceinline__ bool ka_sequence(const KaArgs& a, KaSeq& q) {  // false: nothing to do
  int id = blockIdx.x;
  q.h = id % a.kv_heads;  // eight heads: one per XCD, whose L2 then holds that head's keys
  id /= a.kv_heads;
  if (MANY) {
    q.b = id % a.batch;
    q.block0 = id / a.batch;
    if (a.last_first) q.block0 = a.blocks - 1 - q.block0;
    q.split = 0;
  } else {
    // The blocks of one sequence run next to each other, as they read the same keys (24 sequences of up to 4000 keys with 1 to
    // 200 new tokens, with one term a weight: 168 us block by block, 97 so), and its last ones, which see the most, first
    // (2 x 512 tokens over 4096 keys 102.9 -> 100.3 us, head dim 64 71.0 -> 69.5; those 24 sequences 101 -> 103).
    q.block0 = a.blocks - 1 - id % a.blocks;
    id /= a.blocks;
    q.split = id % a.splits;
    q.b = id / a.splits;
  }
  if (a.longest_first) q.b = ka_longest_first(a, q.b);
  q.G = a.heads / a.kv_heads;
  q.start = a.query_start ? ka_scalar(a.query_start + q.b) : q.b;
  if (q.start < 0 || q.start >= a.tokens) return false;
  q.n_new = min(a.query_start ? ka_scalar(a.query_start + q.b + 1) - q.start : 1, a.tokens - q.start);
  q.rows = q.n_new * q.G;  // (tokens * heads < 2^31, checked by the host)
  q.kv_len = (int)min((long)max(ka_scalar(a.seq_lens + q.b), 0), (long)a.table_width << a.page_shift);
  q.table = a.table + q.b * a.table_stride;
  return true;
}

// The queries of RB blocks of 16 rows from row0 on as second operands: column c = lane % 16 of block rb is row
// row0 + 16 rb + c (past the last row: that one again).  last: the last key each of them sees.
template <int D, int DT, int NQ, int RB>
__device__ __forceinline__ void ka_queries(const KaArgs& a, const KaSeq& q, int row0, v8bf (&qf)[RB][NQ][D / 32], int (&last)[RB]) {
  typedef typename KaT<DT>::T T;
  typedef T Tv __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int r16 = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(row0 + 16 * rb + r16, q.rows - 1);
    const int i = (unsigned)row / (unsigned)q.G, hq = q.h * q.G + row - i * q.G;
    last[rb] = a.causal ? q.kv_len - q.n_new + i : q.kv_len - 1;
    const T* qp = (const T*)a.q + (q.start + i) * a.q_token_stride + hq * a.q_head_stride + D / 4 * g;
#pragma unroll
    for (int m = 0; m < D / 32; ++m) {
      const Tv raw = *(const Tv*)(qp + 8 * m);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        __bf16 t[NQ];
        // (an infinity becomes NaN: it makes its row that, but every score of it may be minus infinity, as for a row without a key)
        const float f = __builtin_fmaf((float)raw[e], 0.f, (float)raw[e]);
        ka_terms<NQ>(a.negate ? -f : f, t);
#pragma unroll
        for (int n = 0; n < NQ; ++n) qf[rb][n][m][e] = t[n];
      }
    }
  }
}

// Rows in blocks of 16 RB; the waves of the workgroup take key tiles in turn and join what they have at the end.
// What bounds it: the vector pipes (codes to bf16, softmax) in 60 to 73 % of the busy cycles, next to memory.  32 sequences of
// up to 32768 keys, 8 heads of 128, 8 query heads each: 117 us, 5.0 TB/s; 64 sequences x 32 heads of 64, up to 2048 keys: 37.
template <int D, int NW>
struct KaFewLds {
  float joint[NW][16][D + 4];  // (padded rows)
  float stat_m[NW][16], stat_l[NW][16];
};
template <int D, int DT, int NQ, int NP, int RB, int NW, int TB>
__device__ __forceinline__ void ka_few(const KaArgs& a, const KaSeq& q, KaFewLds<D, NW>& lds) {
  typedef typename KaT<DT>::T T;
  constexpr bool NT = RB == 1;
  constexpr int DG = D / 4;    // elements of a key per lane
  constexpr int KM = DG / 8;   // MFMAs per 16 keys = dwords of a key per lane
  constexpr int PB = D / 32;   // bytes of a piece = scales of a token = dwords of values per lane and 16 keys
  constexpr int VJ = D / 16;   // MFMAs of the second product
  constexpr int TK = 16 * TB;  // keys of a tile
  auto& joint = lds.joint;
  auto& stat_m = lds.stat_m;
  auto& stat_l = lds.stat_l;
  const int h = q.h, split = q.split, block0 = q.block0, G = q.G, start = q.start, n_new = q.n_new, rows = q.rows, kv_len = q.kv_len;
  const int* table = q.table;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pm = (1 << a.page_shift) - 1;

  // where this lane's share of 16 keys lies
  const uint32_t kc_off = r16 * (D / 2) + g * (DG / 2), vc_off = (g * 16 + r16) * (4 * PB);
  const uint32_t ks_off = r16 * PB + (D == 64 ? g >> 1 : D == 128 ? g : 2 * g), vs_off = (g * PB + r16 / (512 / D)) * 4;

  for (int row0 = block0 * 16 * RB; row0 < rows; row0 += a.blocks * 16 * RB) {
    const int i_first = (unsigned)row0 / (unsigned)G, i_last = (unsigned)(min(row0 + 16 * RB, rows) - 1) / (unsigned)G;
    const int see_all = a.causal ? kv_len - n_new + i_first : kv_len - 1;            // last key every row sees
    const int n_keys = a.causal ? max(kv_len - n_new + i_last + 1, 0) : kv_len;      // keys any row sees
    const int tiles = (n_keys + TK - 1) / TK;
    const int piece = max((tiles + a.splits - 1) / a.splits, a.splits > 1 ? KA_PIECE / TK : 1);
    const int t_begin = min(split * piece, tiles), t_end = min(t_begin + piece, tiles);

    v8bf qf[RB][NQ][KM];
    int last[RB];
    ka_queries<D, DT, NQ, RB>(a, q, row0, qf, last);

    v4f o[RB][VJ];
    float mx[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      mx[rb] = KA_M0;
      l[rb] = 0.f;
#pragma unroll
      for (int j = 0; j < VJ; ++j) o[rb][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    }

    // ---- tiles on their way: pages first, then codes and scales.  Every load is in range whatever the tables hold:
    // blocks past the last key are the last block, a page that does not exist is page 0, and both are masked.
    struct Tile {
      uint32_t k[TB][KM], v[TB][PB], ks[TB], vs[TB];
      uint32_t nan_at;  // values of this lane (bit 4 tb + i) that are NaN in a tile with a mask
      uint32_t there;
    };
    const int last_block = (n_keys - 1) >> 4;
    auto page_of = [&](int t, int tb) { return ka_scalar(table + (min(TB * t + tb, last_block) >> (a.page_shift - 4))); };
    auto load = [&](Tile& x, int t, const int(&pages)[TB]) {
      x.there = 0;
      x.nan_at = 0;
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        int page = pages[tb];
        const bool ok = (unsigned)page < (unsigned)a.pages;
        page = ok ? page : 0;
        x.there |= (uint32_t)ok << tb;
        const long at = (((long)page * a.kv_heads + h) << a.page_shift) + ((min(TB * t + tb, last_block) << 4) & pm);
        const uint8_t* kc = a.kc + at * (D / 2);  // (uniform bases, 32-bit offsets per lane)
        const uint8_t* vc = a.vc + at * (D / 2);
        if (KM == 2) {
          const v2i u = ka_codes<NT>((const v2i*)(kc + kc_off));
          x.k[tb][0] = u[0], x.k[tb][1] = u[1];
        } else {
#pragma unroll
          for (int m = 0; m < KM; m += 4) {
            const v4i u = ka_codes<NT>((const v4i*)(kc + kc_off + 4 * m));
            x.k[tb][m] = u[0], x.k[tb][m + 1] = u[1], x.k[tb][m + 2] = u[2], x.k[tb][m + 3] = u[3];
          }
        }
        const uint8_t* ks = a.ks + at * PB;
        if (D == 256) x.ks[tb] = *(const uint16_t*)(ks + ks_off);
        else x.ks[tb] = ks[ks_off];
        if (PB == 2) {
          const v2i u = ka_codes<NT>((const v2i*)(vc + vc_off));
          x.v[tb][0] = u[0], x.v[tb][1] = u[1];
        } else {
#pragma unroll
          for (int m = 0; m < PB; m += 4) {
            const v4i u = ka_codes<NT>((const v4i*)(vc + vc_off + 4 * m));
            x.v[tb][m] = u[0], x.v[tb][m + 1] = u[1], x.v[tb][m + 2] = u[2], x.v[tb][m + 3] = u[3];
          }
        }
        x.vs[tb] = *(const uint32_t*)(a.vs + at * PB + vs_off);
      }
    };

    v4f s[RB][TB];
    auto scores = [&](const Tile& x, v4f(&to)[RB][TB]) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        v8bf kf[KM];
#pragma unroll
        for (int m = 0; m < KM; ++m) {
          const float sc = kv4_scale_of(x.ks[tb], D == 256 && m >= KM / 2 ? 1 : 0);
          v4i u;
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = (int)ka_pair(x.k[tb][m], sc, e);
          kf[m] = __builtin_bit_cast(v8bf, u);
        }
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
    auto mask = [&](Tile& x, v4f(&to)[RB][TB], int t) {
      if (TK * t + TK - 1 > see_all || x.there != (1u << TB) - 1) {
        HX_OPAQUE_V(x.nan_at);  // keeps this a branch: as selects the masks would cost every tile as much as the softmax
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (TK * t + 16 * tb + 4 * g + e > last[rb] || !((x.there >> tb) & 1)) to[rb][tb][e] = -INFINITY;
        // A masked p is zero, but zero times NaN is not: the scales behind the last key (memory that nobody has written, or
        // another sequence's) become small finite ones, and the NaN that a row does see is put in after the product.
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = TK * t + 16 * tb + 4 * g + i < n_keys && ((x.there >> tb) & 1);
            const bool nan = ((x.vs[tb] >> (8 * i)) & 255) == 255;
            if (!there || nan) x.vs[tb] = (x.vs[tb] & ~(255u << (8 * i))) | (1u << (8 * i));
            if (there && nan) x.nan_at |= 1u << (4 * tb + i);
          }
      }
    };
    // Moves the reference points where a score lies far above.  The four lanes that share a column agree on its point.
    auto vote = [&]() {
      float top[RB];
      bool far = false;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        top[rb] = s[rb][0][0];
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[rb] = fmaxf(top[rb], s[rb][tb][e]);
        top[rb] *= a.c;
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
    auto weights = [&](v8bf(&pf)[RB][NP], int half) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][2 * half + tb][e], a.c, -mx[rb]));
            l[rb] += p;
            __bf16 u[NP];
            ka_terms<NP>(p, u);
#pragma unroll
            for (int n = 0; n < NP; ++n) pf[rb][n][4 * tb + e] = u[n];
          }
    };
    auto values = [&](const Tile& x, const v8bf(&pf)[RB][NP], int half) {
      // byte jj of a piece is elements 2jj, 2jj+1 of it; eight tokens, regrouped by element
      float sv[2][4];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[tb][i] = kv4_scale_of(x.vs[2 * half + tb], i);
#pragma unroll
      for (int jj = 0; jj < VJ / 2; ++jj) {
        uint32_t u[8];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int byte = i * PB + jj;
            u[4 * tb + i] = ka_pair(x.v[2 * half + tb][byte / 4], sv[tb][i], byte % 4);
          }
        v4i even, odd;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          even[e] = (int)__builtin_amdgcn_perm(u[2 * e + 1], u[2 * e], 0x05040100);
          odd[e] = (int)__builtin_amdgcn_perm(u[2 * e + 1], u[2 * e], 0x07060302);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int n = NP - 1; n >= 0; --n) {
            o[rb][2 * jj] = Mfma16<true>::run16(__builtin_bit_cast(v8bf, even), pf[rb][n], o[rb][2 * jj]);
            o[rb][2 * jj + 1] = Mfma16<true>::run16(__builtin_bit_cast(v8bf, odd), pf[rb][n], o[rb][2 * jj + 1]);
          }
      }
    };
    auto put_nan = [&](const Tile& x, int t) {
      if (__builtin_amdgcn_ballot_w64(x.nan_at != 0) != 0) {
        // rows of the count: pieces; a piece lies in one block, so all of it is NaN for the queries that see the token
#pragma unroll
        for (int half = 0; half < TB / 2; ++half) {
          v8bf bad;
#pragma unroll
          for (int e = 0; e < 8; ++e) bad[e] = (x.nan_at >> (8 * half + e)) & 1 ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            v8bf sees;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sees[e] = TK * t + 16 * (2 * half + (e >> 2)) + 4 * g + (e & 3) <= last[rb] ? (__bf16)1.f : (__bf16)0.f;
            const v4f count = Mfma16<true>::run16(bad, sees, (v4f){0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int j = 0; j < VJ; ++j)
                if (count[e] > 0.f) o[rb][j][e] = __builtin_nanf("");
          }
        }
      }
    };

    if (t_begin + w < t_end) {
      // The loads run one tile ahead, the pages of the next one already known; past the last tile that one again, so that
      // every step issues the same loads and the waits are for the older tile alone.
      const int t_last = t_end - 1;
      Tile ring[2];
      int t = t_begin + w, t1 = min(t + NW, t_last), pages[TB];
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) pages[tb] = page_of(t, tb);
      load(ring[0], t, pages);
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) pages[tb] = page_of(t1, tb);
      auto step = [&](Tile& cur, Tile& next) {
        load(next, t1, pages);
        t1 = min(t + 2 * NW, t_last);
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) pages[tb] = page_of(t1, tb);
        scores(cur, s);
        mask(cur, s, t);
        vote();
#pragma unroll
        for (int half = 0; half < TB / 2; ++half) {
          v8bf pf[RB][NP];
          weights(pf, half);
          values(cur, pf, half);
        }
        put_nan(cur, t);
        t += NW;
      };
      for (;;) {
        step(ring[0], ring[1]);
        if (t >= t_end) break;
        step(ring[1], ring[0]);
        if (t >= t_end) break;
      }
    }

    // ---- join the waves: element d = (4g + e) * D/16 + j of query c is o[j][e] of lane (c, g)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float lt = l[rb] + __shfl_xor(l[rb], 16);
      lt += __shfl_xor(lt, 32);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < VJ; j += 4)
          *(v4f*)&joint[w][r16][(4 * g + e) * VJ + j] = (v4f){o[rb][j][e], o[rb][j + 1][e], o[rb][j + 2][e], o[rb][j + 3][e]};
      if (g == 0) stat_m[w][r16] = mx[rb], stat_l[w][r16] = lt;
      __syncthreads();
      for (int at = tid; at < 16 * (D / 4); at += NW * 64) {
        const int c = at / (D / 4), d = at % (D / 4) * 4;
        const int row = row0 + 16 * rb + c;
        if (row < rows) {
          float top = stat_m[0][c];
#pragma unroll
          for (int v = 1; v < NW; ++v) top = fmaxf(top, stat_m[v][c]);
          float sum = 0.f;
          v4f acc = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < NW; ++v) {
            const float f = __builtin_amdgcn_exp2f(stat_m[v][c] - top);
            sum += stat_l[v][c] * f;
            acc += *(const v4f*)&joint[v][c][d] * f;
          }
          const int i = (unsigned)row / (unsigned)G, hq = h * G + row - i * G;
          const long to = (long)(start + i) * a.heads + hq;
          if (a.splits == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key gives zeros
            typedef T Tv __attribute__((ext_vector_type(4)));
            Tv v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(acc[e] * inv);
            *(Tv*)((T*)a.out + to * D + d) = v;
          } else {
            *(v4f*)(a.part_o + (to * a.splits + split) * D + d) = acc;
            if (d == 0) *(v2f*)(a.part_ml + (to * a.splits + split) * 2) = (v2f){top, sum};
          }
        }
      }
      __syncthreads();
    }
  }
}

template <int D, int DT, int NQ, int NP, int RB, int NW, int TB>
__global__ __launch_bounds__(NW * 64, RB > 1 || D > 128 || DT == HX_F32 ? 2 : D == 64 ? 4 : DT == HX_BF16 ? 3 : 2) void hx_kv4_attention_kernel(KaArgs a) {
  __shared__ __attribute__((aligned(16))) KaFewLds<D, NW> lds;
  KaSeq q;
  if (ka_sequence<false>(a, q)) ka_few<D, DT, NQ, NP, RB, NW, TB>(a, q, lds);
}

#include "kv4_attention_rows.h"

// Joins the splits of a row: four waves per row take every fourth split, four at a time; lane i of a wave holds the
// statistics of split i.
#define KA_MOST 64  // splits of a row at most
template <int D, int DT>
__global__ __launch_bounds__(256) void hx_kv4_attention_join(KaArgs a) {
  typedef typename KaT<DT>::T T;
  constexpr int E = D / 64;
  __shared__ float part[4][D];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  for (long row = blockIdx.x; row < (long)a.tokens * a.heads; row += gridDim.x) {
    const int t = (unsigned)row / (unsigned)a.heads;  // (row < 2^31)
    if (a.query_start && (t < a.query_start[0] || t >= a.query_start[a.batch])) continue;  // behind the last sequence
    const float* ml = a.part_ml + row * a.splits * 2;
    const bool there = lane < a.splits;
    float l = there ? ml[2 * lane + 1] : 0.f;
    const float m = there ? ml[2 * lane] : KA_M0;
    float top = m;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - top);  // (a split without keys has written nothing else)
    float sum = l * f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    const float* o = a.part_o + row * a.splits * D + lane * E;
    for (int s0 = w; s0 < a.splits; s0 += 16) {
      float v[4][E];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] = o[(long)min(s0 + 4 * i, a.splits - 1) * D + e];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + 4 * i;
        const float fs = __shfl(f, s & 63);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (s < a.splits && fs != 0.f) acc[e] += v[i][e] * fs;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) part[w][lane * E + e] = acc[e];
    __syncthreads();
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int d = threadIdx.x; d < D; d += 256) ((T*)a.out)[row * D + d] = (T)((part[0][d] + part[1][d] + part[2][d] + part[3][d]) * inv);
    __syncthreads();
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct KaPlan {
  int rb, nw, blocks, splits;
  bool many;  // hx_kv4_attention_rows
};

static KaPlan ka_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t max_query, int64_t max_keys, int dt) {
  KaPlan p;
  // (a max_query that is padded, for a graph or by a server's limit, plans what the tokens need)
  const int64_t rows = (max_query < tokens ? max_query : tokens) * (heads / kv_heads);
  // Two blocks of rows share a conversion of the keys and values.  A head dim of 256 leaves no registers for it (680 to 1640
  // bytes of scratch a lane; 512 tokens over 4096 keys, bf16: 123 us with one block, 391 with two), nor does an fp32 query at
  // 128 (196 bytes; 91 and 97); at 64, where it would give a tenth (61 and 55), fp32 goes the same way.
  p.rb = rows > 16 && D <= 128 && dt != HX_F32 ? 2 : 1;
  p.nw = 4;
  p.many = false;
  // 128 rows per workgroup with the conversion shared, or 32 with the keys divided among the waves: both run two workgroups
  // per compute unit; in units of time, the former takes 45 for as many keys as the latter takes 12 for, in whole rounds (its
  // workgroups end together), the latter in as many rounds as it takes.  bf16, 32 heads of 128 on 8: 8 x 512 tokens over 2048
  // keys 183 and 203 us, 4 x 1024 over 4096 345 and 361, 2048 over 10240 438 both; but 12 x 200 over 4000 280 and 243, 2 x 512
  // over 4096 137 and 103.
  if (p.rb == 2 && rows > 64) {
    const int64_t slots = 2 * hx_cu_count(), pairs = batch * kv_heads;
    const int64_t many = (pairs * ((rows + KR_ROWS - 1) / KR_ROWS) + slots - 1) / slots * slots * 45, few = pairs * ((rows + 31) / 32) * 12;
    p.many = many < few;
  }
  const int64_t per = p.many ? KR_ROWS : 16 * p.rb;
  int64_t blocks = (rows + per - 1) / per;
  if (blocks < 1) blocks = 1;
  if (blocks > 65536) blocks = 65536;
  while (blocks > 1 && kv_heads * blocks > KA_GRID) blocks /= 2;
  p.blocks = (int)blocks;
  // Keys are split, into pieces of at least 1024, until there are sixteen workgroups per compute unit (sequences differ in
  // length, and what ends last counts) or two of the larger ones; a sequence shorter than the table's width uses fewer.
  // Where there are four per unit without a split the joining costs more than it gives (64 sequences x 32 heads of up to
  // 2048 keys: 42 us whole, 48 in two pieces).  One sequence of 32768 keys, 8 heads: pieces of 2048 18.4 us, 1024 14.0,
  // 512 15.2; 32 sequences up to 32768: 122, 124, 125; 4 new tokens of 16 sequences of 8192: two per unit 46, four 51.
  // Where there are four per unit, one much longer sequence is not split either: 128 sequences of 500 keys, 8 heads, one of
  // 32768 among them take 169 us, most of it that one.
  const int64_t base = batch * kv_heads * blocks, cus = hx_cu_count(), most = max_keys / KA_PIECE;
  const int64_t want = base >= 4 * cus || p.many ? 1 : ((p.rb == 1 ? 16 : 2) * cus + base - 1) / base;
  int64_t s = want < most ? want : most;
  p.splits = (int)(s < 1 ? 1 : s > KA_MOST ? KA_MOST : s);
  return p;
}

static int ka_check_sizes(const char* who, int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t page, int64_t width,
                          int64_t max_query, int dt) {
  if (tokens < 0 || batch < 0 || heads < 0 || width < 0 || max_query < 0) {
    hx_set_error("%s: negative size", who);
    return HX_ERR_BAD_ARG;
  }
  if (kv_heads < 1 || heads % kv_heads != 0) {
    hx_set_error("%s: %lld query heads do not divide by %lld key/value heads", who, (long long)heads, (long long)kv_heads);
    return HX_ERR_BAD_ARG;
  }
  if (dt != HX_F16 && dt != HX_BF16 && dt != HX_F32) {
    hx_set_error("%s: dtype must be HX_F16, HX_BF16 or HX_F32, got %d", who, dt);
    return HX_ERR_BAD_ARG;
  }
  if (tokens * heads >= (1l << 31) - 4096 || tokens > (1l << 30) || heads > 65535 || batch > (1l << 24) || width * page >= (1l << 31) - 64 || batch * kv_heads > (1l << 30)) {
    hx_set_error("%s: too many tokens, sequences or keys", who);
    return HX_ERR_UNSUPPORTED;
  }
  return 0;
}

extern "C" size_t hx_kv4_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t page,
                                                   int64_t table_width, int64_t max_query, int dtype) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0) return 0;
  const KaPlan p = ka_plan(tokens, batch, heads, kv_heads, D, max_query, table_width * page, dtype);
  return p.splits == 1 ? 0 : (size_t)tokens * heads * p.splits * (D + 2) * sizeof(float);
}

extern "C" int hx_kv4_attention_path(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t page,
                                     int64_t table_width, int64_t max_query, int dtype) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0) return 0;
  const KaPlan p = ka_plan(tokens, batch, heads, kv_heads, D, max_query, table_width * page, dtype);
  return (p.many ? 3 : p.rb) + (p.splits > 1 ? 8 : 0);
}

template <int D, int DT>
static void ka_launch(const KaArgs& a, const KaPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.kv_heads * a.batch * p.splits * p.blocks)), block(p.nw * 64);  // (at most KA_GRID)
  constexpr int NQ = DT == HX_BF16 ? 1 : DT == HX_F16 ? 2 : 3, NP = DT == HX_F32 ? 3 : 2;
  if (p.many) {
    if constexpr (D <= 128 && DT != HX_F32) hx_launch(hx_kv4_attention_rows<D, DT, NQ, NP>, grid, dim3(KR_WAVES * 64), 0, s, a);
  } else if (p.rb == 1) {
    hx_launch(hx_kv4_attention_kernel<D, DT, NQ, NP, 1, 4, 2>, grid, block, 0, s, a);
  } else if constexpr (D <= 128 && DT != HX_F32) {
    hx_launch(hx_kv4_attention_kernel<D, DT, NQ, NP, 2, 4, 2>, grid, block, 0, s, a);
  }
  if (p.splits > 1) hx_launch(hx_kv4_attention_join<D, DT>, dim3((unsigned)min((long)a.tokens * a.heads, KA_GRID)), dim3(256), 0, s, a);
}

extern "C" int hx_kv4_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_codes, const void* k_scales,
                                const void* v_codes, const void* v_scales, const int32_t* block_table, int64_t table_stride,
                                const int32_t* seq_lens, const int32_t* query_start, void* out, int64_t tokens, int64_t batch,
                                int64_t heads, int64_t kv_heads, int64_t D, int64_t pages, int64_t page, int64_t table_width,
                                int64_t max_query, float scale, int causal, int dtype, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* who = "hx_kv4_attention";
  int rc = kv4_check_cache(who, k_codes, k_scales, v_codes, v_scales, pages, page, kv_heads, D);
  if (rc == 0) rc = ka_check_sizes(who, tokens, batch, heads, kv_heads, page, table_width, max_query, dtype);
  if (rc != 0 || tokens == 0 || batch == 0 || heads == 0) return rc;
  if (!q || !out || !seq_lens || (table_width > 0 && !block_table)) {
    hx_set_error("%s: null pointer", who);
    return HX_ERR_BAD_ARG;
  }
  if (!query_start && tokens != batch) {
    hx_set_error("%s: without query_start there is one token for each of the %lld sequences, got %lld", who, (long long)batch, (long long)tokens);
    return HX_ERR_BAD_ARG;
  }
  if (batch > 1 && table_stride < table_width) {
    hx_set_error("%s: page table rows overlap", who);
    return HX_ERR_BAD_ARG;
  }
  if (((uintptr_t)q & (dtype == HX_F32 ? 3 : 1)) || ((uintptr_t)out & 15) ||
      (((uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)query_start) & 3)) {
    hx_set_error("%s: out must be 16-byte aligned, the other pointers aligned to their elements", who);
    return HX_ERR_UNSUPPORTED;
  }
  const KaPlan p = ka_plan(tokens, batch, heads, kv_heads, D, query_start ? max_query : 1, table_width * page, dtype);
  const size_t need = p.splits == 1 ? 0 : (size_t)tokens * heads * p.splits * (D + 2) * sizeof(float);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    hx_set_error("%s: workspace must be 16-byte aligned and at least %zu bytes (got %zu)", who, need, workspace_bytes);
    return HX_ERR_WORKSPACE;
  }
  KaArgs a;
  a.q = q, a.q_token_stride = q_token_stride, a.q_head_stride = q_head_stride, a.out = out;
  a.kc = (const uint8_t*)k_codes, a.ks = (const uint8_t*)k_scales, a.vc = (const uint8_t*)v_codes, a.vs = (const uint8_t*)v_scales;
  a.table = block_table, a.table_stride = table_stride, a.seq_lens = seq_lens, a.query_start = query_start;
  a.part_o = (float*)workspace, a.part_ml = need ? a.part_o + (size_t)tokens * heads * p.splits * D : nullptr;
  a.negate = scale < 0.f;
  a.c = fmaxf(fabsf(scale) * 1.44269504f, 1e-37f);  // (zero times a masked score would be NaN)
  a.tokens = (int)tokens, a.batch = (int)batch, a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.pages = (int)pages;
  a.page_shift = __builtin_ctzll((unsigned long long)page), a.table_width = pages > 0 ? (int)table_width : 0, a.causal = causal != 0;
  a.splits = p.splits, a.blocks = p.blocks;
  // Workgroups of 128 rows in more than one round: the last blocks see the most keys and go first (4096 tokens over 4096
  // keys 241 -> 210 us); in one round they start together, and the first ones first is better (2048 over 10240 460 and 440 us).
  const int64_t groups = batch * kv_heads * p.blocks * p.splits;
  a.longest_first = batch > 1 && groups > 2 * hx_cu_count();
  a.len_shift = 0;
  while (((table_width * page) >> a.len_shift) > 255) ++a.len_shift;
  a.last_first = p.many && groups > 2 * hx_cu_count();
  auto go = [&](auto dc) {
    constexpr int DC = decltype(dc)::value;
    if (dtype == HX_F16) ka_launch<DC, HX_F16>(a, p, (hipStream_t)stream);
    else if (dtype == HX_BF16) ka_launch<DC, HX_BF16>(a, p, (hipStream_t)stream);
    else ka_launch<DC, HX_F32>(a, p, (hipStream_t)stream);
  };
  // as many sequences in a launch as it has room for (so many that their keys are not split)
  const int64_t room = KA_GRID / (kv_heads * p.blocks * p.splits), es = dtype == HX_F32 ? 4 : 2;
  for (int64_t b = 0; b < batch; b += room) {
    a.batch = (int)(batch - b < room ? batch - b : room);
    a.table = block_table + b * table_stride, a.seq_lens = seq_lens + b;
    if (query_start) {
      a.query_start = query_start + b;
    } else {
      a.q = (const char*)q + b * q_token_stride * es, a.out = (char*)out + b * heads * D * es;
      a.tokens = a.batch;
    }
    if (D == 64) go(std::integral_constant<int, 64>{});
    else if (D == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
  }
  const hipError_t e = hx_launch_status();
  if (e != hipSuccess) {
    hx_set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}
