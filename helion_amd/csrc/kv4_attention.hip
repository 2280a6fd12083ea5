// Attention over the 4-bit key/value cache (format and layout: kv4_format.h), for new tokens of many sequences at once:
//   out[t, hq] = sum_j p_j v[j, hq / G] / sum_j p_j,   p_j = 2^(c (q[t, hq] . k[j, hq / G]) - m),  c = scale * log2(e)
// over the keys j the token may see, in one pass with a running reference point m and sum.  G = query heads per key/value
// head; the keys of sequence b are the first seq_lens[b] slots of its row of the page table.
//
// Precision: an e2m1 value times a power of two is a bf16 number, so keys and values enter the matrix instructions
// exactly.  The other operand of each product is a sum of bf16 terms: one for a bf16 query, two for fp16 (11 bits fit in
// 16), three for fp32; p as two terms (2^-17 of it is lost) or three for fp32, or as one where a comment says so.  Products are
// summed in fp32, as are the statistics.
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
  float c;         // softmax scale * log2(e)
  int tokens, batch, heads, kv_heads, pages, page_shift, table_width, causal, splits, blocks;
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

// f = t[0] + t[1] + .. + t[N-1] with bf16 terms, each the rounding of what the ones before it leave
template <int N>
__device__ __forceinline__ void ka_terms(float f, __bf16 (&t)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    t[n] = (__bf16)f;
    f -= (float)t[n];
  }
}

template <int D, int DT, int NQ, int NP, int RB, int NW>
__global__ __launch_bounds__(NW * 64) void hx_kv4_attention_kernel(KaArgs a) {
  typedef typename KaT<DT>::T T;
  constexpr int DG = D / 4;    // elements of a key per lane
  constexpr int KM = DG / 8;   // MFMAs per 16 keys = dwords of a key per lane
  constexpr int PB = D / 32;   // bytes of a piece = scales of a token = dwords of values per lane and 16 keys
  constexpr int VJ = D / 16;   // MFMAs of the second product
  constexpr int OSTR = D + 4;  // row stride of the joining buffer, in floats
  __shared__ __attribute__((aligned(16))) float joint[NW][16][OSTR];
  __shared__ float stat_m[NW][16], stat_l[NW][16];

  int id = blockIdx.x;
  const int h = id % a.kv_heads;  // eight heads: one per XCD, whose L2 then holds that head's keys
  id /= a.kv_heads;
  const int b = id % a.batch;
  id /= a.batch;
  const int split = id % a.splits;
  const int block0 = id / a.splits;

  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.heads / a.kv_heads;
  const int start = a.query_start ? a.query_start[b] : b;
  int n_new = a.query_start ? a.query_start[b + 1] - start : 1;
  if (start < 0 || start >= a.tokens) return;
  n_new = min(n_new, a.tokens - start);
  const int pm = (1 << a.page_shift) - 1;
  const int kv_len = (int)min((long)max(a.seq_lens[b], 0), (long)a.table_width << a.page_shift);
  const int* table = a.table + b * a.table_stride;
  const long rows = (long)n_new * G;

  for (long block = block0; block * (16 * RB) < rows; block += a.blocks) {
    const long row0 = block * (16 * RB);
    const int i_first = (int)(row0 / G), i_last = (int)((min(row0 + 16 * RB, rows) - 1) / G);
    const int see_all = a.causal ? kv_len - n_new + i_first : kv_len - 1;            // last key every row sees
    const int n_keys = a.causal ? max(kv_len - n_new + i_last + 1, 0) : kv_len;      // keys any row sees
    const int tiles = (n_keys + 31) >> 5;
    const int t_begin = (int)((long)tiles * split / a.splits), t_end = (int)((long)tiles * (split + 1) / a.splits);

    // ---- this wave's queries: column c = lane % 16 of block rb is row row0 + 16 rb + c
    v8bf qf[RB][NQ][KM];
    int last[RB];  // the last key the row sees
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const long row = row0 + 16 * rb + r16;
      const int i = (int)(min(row, rows - 1) / G), hq = h * G + (int)(min(row, rows - 1) - (long)i * G);
      last[rb] = a.causal ? kv_len - n_new + i : kv_len - 1;
      const T* qp = (const T*)a.q + (start + i) * a.q_token_stride + hq * a.q_head_stride + DG * g;
      typedef T Tv __attribute__((ext_vector_type(8), aligned(sizeof(T))));
#pragma unroll
      for (int m = 0; m < KM; ++m) {
        const Tv raw = *(const Tv*)(qp + 8 * m);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          __bf16 t[NQ];
          ka_terms<NQ>((float)raw[e], t);
#pragma unroll
          for (int n = 0; n < NQ; ++n) qf[rb][n][m][e] = t[n];
        }
      }
    }

    v4f o[RB][VJ];
    float mx[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      mx[rb] = KA_M0;
      l[rb] = 0.f;
#pragma unroll
      for (int j = 0; j < VJ; ++j) o[rb][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    }

    // ---- a tile on its way: pages first, then codes and scales, one step ahead of their use.  Every load is in range
    // whatever the tables hold: blocks past the last key are the last block, a page that does not exist is page 0, and
    // both are masked.
    struct Tile {
      uint32_t k[2][KM], v[2][PB], ks[2], vs[2];
      int there;
    };
    const int last_block = (n_keys - 1) >> 4;
    auto page_of = [&](int t, int tb) { return table[min(2 * t + tb, last_block) >> (a.page_shift - 4)]; };
    auto load = [&](Tile& x, int t, int page0, int page1) {
      x.there = 0;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        int page = tb ? page1 : page0;
        const bool ok = (unsigned)page < (unsigned)a.pages;
        page = ok ? page : 0;
        x.there |= ok << tb;
        const long at = (((long)page * a.kv_heads + h) << a.page_shift) + ((min(2 * t + tb, last_block) << 4) & pm);
        const uint8_t* kc = a.kc + at * (D / 2) + r16 * (D / 2) + g * (DG / 2);
        const uint8_t* vc = a.vc + at * (D / 2) + (g * 16 + r16) * (4 * PB);
        if (KM == 2) {
          const v2i u = *(const v2i*)kc;
          x.k[tb][0] = u[0], x.k[tb][1] = u[1];
        } else {
#pragma unroll
          for (int m = 0; m < KM; m += 4) {
            const v4i u = *(const v4i*)(kc + 4 * m);
            x.k[tb][m] = u[0], x.k[tb][m + 1] = u[1], x.k[tb][m + 2] = u[2], x.k[tb][m + 3] = u[3];
          }
        }
        if (PB == 2) {
          const v2i u = *(const v2i*)vc;
          x.v[tb][0] = u[0], x.v[tb][1] = u[1];
        } else {
#pragma unroll
          for (int m = 0; m < PB; m += 4) {
            const v4i u = *(const v4i*)(vc + 4 * m);
            x.v[tb][m] = u[0], x.v[tb][m + 1] = u[1], x.v[tb][m + 2] = u[2], x.v[tb][m + 3] = u[3];
          }
        }
        const uint8_t* ks = a.ks + at * PB + r16 * PB;
        if (D == 64) x.ks[tb] = ks[g >> 1];
        else if (D == 128) x.ks[tb] = ks[g];
        else x.ks[tb] = *(const uint16_t*)(ks + 2 * g);
        x.vs[tb] = *(const uint32_t*)(a.vs + at * PB + (g * PB + r16 / (512 / D)) * 4);
      }
    };

    auto multiply = [&](const Tile& x, int t) {
      // scores
      v4f s[RB][2];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        v8bf kf[KM];
#pragma unroll
        for (int m = 0; m < KM; ++m) {
          const float sc = kv4_scale(D == 256 ? (m < KM / 2 ? x.ks[tb] & 255 : x.ks[tb] >> 8) : x.ks[tb]);
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
          s[rb][tb] = acc * a.c;
        }
      }
      uint32_t vs[2] = {x.vs[0], x.vs[1]};
      uint32_t nan_at = 0;  // values of this lane (bit 4 tb + i) that are NaN in a tile with a mask
      if (32 * t + 31 > see_all || x.there != 3) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (32 * t + 16 * tb + 4 * g + e > last[rb] || !((x.there >> tb) & 1)) s[rb][tb][e] = -INFINITY;
        // A masked p is zero, but zero times NaN is not: the scales behind the last key (memory that nobody has written, or
        // another sequence's) become small finite ones, and the NaN that a row does see is put in after the product.
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = 32 * t + 16 * tb + 4 * g + i < n_keys && ((x.there >> tb) & 1);
            const bool nan = ((x.vs[tb] >> (8 * i)) & 255) == 255;
            if (!there || nan) vs[tb] = (vs[tb] & ~(255u << (8 * i))) | (1u << (8 * i));
            if (there && nan) nan_at |= 1u << (4 * tb + i);
          }
      }
      // softmax: the reference point of a row is the same in the four lanes that share its column
      v8bf pf[RB][NP];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float top = fmaxf(fmaxf(fmaxf(s[rb][0][0], s[rb][0][1]), fmaxf(s[rb][0][2], s[rb][0][3])),
                          fmaxf(fmaxf(s[rb][1][0], s[rb][1][1]), fmaxf(s[rb][1][2], s[rb][1][3])));
        if (__builtin_amdgcn_ballot_w64(top > mx[rb] + KA_STEP) != 0) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float next = fmaxf(mx[rb], top), f = __builtin_amdgcn_exp2f(mx[rb] - next);
          mx[rb] = next;
          l[rb] *= f;
#pragma unroll
          for (int j = 0; j < VJ; ++j) o[rb][j] *= f;
        }
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(s[rb][tb][e] - mx[rb]);
            l[rb] += p;
            __bf16 u[NP];
            ka_terms<NP>(p, u);
#pragma unroll
            for (int n = 0; n < NP; ++n) pf[rb][n][4 * tb + e] = u[n];
          }
      }
      // values: byte jj of a piece is elements 2jj, 2jj+1 of it; eight tokens, regrouped by element
      float sv[2][4];
#pragma unroll
      for (int tb = 0; tb < 2; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[tb][i] = kv4_scale((vs[tb] >> (8 * i)) & 255);
#pragma unroll
      for (int jj = 0; jj < VJ / 2; ++jj) {
        uint32_t u[8];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int byte = i * PB + jj;
            u[4 * tb + i] = ka_pair(x.v[tb][byte / 4], sv[tb][i], byte % 4);
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
      if (__builtin_amdgcn_ballot_w64(nan_at != 0) != 0) {
        // rows of the count: pieces; a piece lies in one block, so all of it is NaN for the queries that see the token
        v8bf bad;
#pragma unroll
        for (int e = 0; e < 8; ++e) bad[e] = (nan_at >> e) & 1 ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          v8bf sees;
#pragma unroll
          for (int e = 0; e < 8; ++e) sees[e] = 32 * t + 16 * (e >> 2) + 4 * g + (e & 3) <= last[rb] ? (__bf16)1.f : (__bf16)0.f;
          const v4f count = Mfma16<true>::run16(bad, sees, (v4f){0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < VJ; ++j)
              if (count[e] > 0.f) o[rb][j][e] = __builtin_nanf("");
        }
      }
    };

    if (t_begin + w < t_end) {
      const int t_last = t_end - 1;
      Tile cur, next;
      int t = t_begin + w;
      load(cur, t, page_of(t, 0), page_of(t, 1));
      int t1 = min(t + NW, t_last);
      int pg0 = page_of(t1, 0), pg1 = page_of(t1, 1);
      for (; t < t_end; t += NW) {
        load(next, t1, pg0, pg1);
        t1 = min(t + 2 * NW, t_last);
        pg0 = page_of(t1, 0), pg1 = page_of(t1, 1);
        multiply(cur, t);
        cur = next;
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
        const long row = row0 + 16 * rb + c;
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
          const int i = (int)(row / G), hq = h * G + (int)(row - (long)i * G);
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

// Joins the splits of a row: one wave per row.
template <int D, int DT>
__global__ __launch_bounds__(256) void hx_kv4_attention_join(KaArgs a) {
  typedef typename KaT<DT>::T T;
  constexpr int E = D / 64;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= (long)a.tokens * a.heads) return;
  const int t = (int)(row / a.heads);
  if (a.query_start && (t < a.query_start[0] || t >= a.query_start[a.batch])) return;  // behind the last sequence
  const float* ml = a.part_ml + row * a.splits * 2;
  float top = KA_M0;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
  float sum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float l = ml[2 * s + 1], f = __builtin_amdgcn_exp2f(ml[2 * s] - top);
    if (l == 0.f) continue;  // a split without keys
    sum += l * f;
    const float* o = a.part_o + (row * a.splits + s) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += o[e] * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < E; ++e) ((T*)a.out)[row * D + lane * E + e] = (T)(acc[e] * inv);
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct KaPlan {
  int rb, nw, blocks, splits;
};

static KaPlan ka_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t max_query, int64_t max_keys, int dt) {
  KaPlan p;
  const int64_t rows = max_query * (heads / kv_heads);
  // Four blocks of rows share a conversion of the keys and values; a head dim of 256 or an fp32 query leaves no registers for it.
  p.rb = rows > 16 && D <= 128 && dt != HX_F32 ? 4 : 1;
  p.nw = p.rb == 1 ? 8 : 4;
  int64_t blocks = (rows + 16 * p.rb - 1) / (16 * p.rb);
  if (blocks < 1) blocks = 1;
  if (blocks > 65536) blocks = 65536;
  while (blocks > 1 && batch * kv_heads * blocks > (1l << 30)) blocks /= 2;
  p.blocks = (int)blocks;
  // Keys are split when the rows give fewer than two workgroups per compute unit, into pieces of at least 512 keys.
  const int64_t base = batch * kv_heads * blocks, want = (2l * hx_cu_count() + base - 1) / base, most = max_keys / 512;
  int64_t s = want < most ? want : most;
  p.splits = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
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
  if (tokens > (1l << 30) || batch > (1l << 24) || width * page >= (1l << 31) - 64 || batch * kv_heads > (1l << 30)) {
    hx_set_error("%s: too many tokens, sequences or keys", who);
    return HX_ERR_UNSUPPORTED;
  }
  return 0;
}

extern "C" size_t hx_kv4_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t D, int64_t page,
                                                   int64_t table_width, int64_t max_query, int dtype) {
  if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0) return 0;
  const KaPlan p = ka_plan(batch, heads, kv_heads, D, max_query, table_width * page, dtype);
  return p.splits == 1 ? 0 : (size_t)tokens * heads * p.splits * (D + 2) * sizeof(float);
}

template <int D, int DT>
static void ka_launch(const KaArgs& a, const KaPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.kv_heads * a.batch * p.splits * p.blocks)), block(p.nw * 64);
  constexpr int NQ = DT == HX_BF16 ? 1 : DT == HX_F16 ? 2 : 3, NP = DT == HX_F32 ? 3 : 2;
  if (p.rb == 1) {
    hx_launch(hx_kv4_attention_kernel<D, DT, NQ, NP, 1, 8>, grid, block, 0, s, a);
  } else if constexpr (D <= 128 && DT != HX_F32) {
    hx_launch(hx_kv4_attention_kernel<D, DT, NQ, NP, 4, 4>, grid, block, 0, s, a);
  }
  if (p.splits > 1) hx_launch(hx_kv4_attention_join<D, DT>, dim3((unsigned)(((long)a.tokens * a.heads + 3) / 4)), dim3(256), 0, s, a);
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
  const KaPlan p = ka_plan(batch, heads, kv_heads, D, query_start ? max_query : 1, table_width * page, dtype);
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
  a.c = scale * 1.44269504f;
  a.tokens = (int)tokens, a.batch = (int)batch, a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.pages = (int)pages;
  a.page_shift = __builtin_ctzll((unsigned long long)page), a.table_width = pages > 0 ? (int)table_width : 0, a.causal = causal != 0;
  a.splits = p.splits, a.blocks = p.blocks;
  auto go = [&](auto dc) {
    constexpr int DC = decltype(dc)::value;
    if (dtype == HX_F16) ka_launch<DC, HX_F16>(a, p, (hipStream_t)stream);
    else if (dtype == HX_BF16) ka_launch<DC, HX_BF16>(a, p, (hipStream_t)stream);
    else ka_launch<DC, HX_F32>(a, p, (hipStream_t)stream);
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else if (D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 256>{});
  const hipError_t e = hx_launch_status();
  if (e != hipSuccess) {
    hx_set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}
