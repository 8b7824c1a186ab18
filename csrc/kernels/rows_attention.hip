// Attention of a block of query rows over paged keys, 8-bit (kv_quant.h) or bf16: decode, prompt portions, and the part of
// a group of decode rows whose keys are in common (a shared prefix, read once for the group).
//
// The rows of one kv head are (token, query head of its G) pairs, token-major: a decode step has G rows a sequence, a
// prompt portion G rows a token, a group of sequences with a common prefix G rows a member. A workgroup takes a block of
// 16 RT rows and a range of keys; its four waves take 32-key tiles of the range in turn, each for all the rows:
//   S^T[16 keys][16 rows] = K Q^T   v_mfma_f32_16x16x32_bf16; K fragments come from the cache as they lie (8-bit codes
//     widened in registers; bf16: whole rows, brought into order through LDS), the key's scale joins softmax's scale afterwards: no rounding but the products' own
//   softmax in base 2 by running maximum. The maximum is only raised (and the accumulators rescaled) when a score passes
//     it by more than 2^8: fp32 sums and bf16 weights are relative, so weights up to 2^8 cost no precision
//   O^T[D][16 rows] += V^T P^T      the same instruction over 32 keys. The S^T accumulators are the P^T fragment where
//     the 8 keys of lane group g are 4 g + {0..3} of both 16-key halves; the cache holds V in that order (bf16: V is
//     turned through LDS). V's scale joins the weight before its rounding to bf16, half a step of 2^-8 at most: the instruction's
//     other operand has to be bf16 too. An output's error, its own rounding's 1.6e-3 in root mean square of itself, becomes 2.0 to
//     2.4e-3 by it (32-bit weights, which would need a second product for their rest, 1.6 to 1.8e-3)
// The waves' states join through LDS, parts of a row's keys through rows_join_kernel: (O / l, log2-sum-exp) in fp32.
//
// Waves share no tile, so the key loop has no barrier, and K / V go from HBM to registers: one tile's loads are on their
// way while another is worked on. Rows without keys give zeros. Keys outside a row's range are never read into its result,
// whatever the cache holds there.
#include <type_traits>

#include "kv_quant.h"

namespace xgk {

constexpr float RAISE = 8.f;          // in base 2
constexpr float LOWEST = -3.4e38f;    // the maximum of no key, below every score's: exp2(LOWEST - any) is 0

// A row's weights are 2^(score - maximum - LIFT): their sum, and theirs times the values, stay below 2^127 for values of any size while
// a wave has up to 2^16 keys 2^RAISE above the maximum (2^24 at it). Where the first keys' values (8-bit: their factors) are below 2^-64,
// LIFT_SMALL: a weight times such a factor would be no normal bf16 number, or its product no normal float. A choice of a row's first
// keys, so it costs nothing in the loop; later values may be as large as 2^50 then.
constexpr float LIFT = 24.f, LIFT_SMALL = -48.f, SMALL = 0x1p-64f;

struct RowsArgs {
  const uint16_t* q;
  int64_t q_stride;
  const uint8_t* k;       // codes, or bf16 rows [num_blocks, Hkv, bs, D]
  const uint8_t* v;
  const float* scales;    // 8-bit
  const int32_t* tables;
  int64_t table_stride;
  int width, num_blocks;
  const int32_t* seq_lens;
  float* part_out;        // [parts, D]; null: whole rows, written to `out`
  float* part_lse;        // [parts]
  uint16_t* out;
  int64_t out_stride;
  int Hq, Hkv, G, bs;
  float scale;            // softmax's, in base 2
  uint32_t page_magic;    // page_of
  int least;              // decode: units of 128 keys that a share has where there are that many
};

// tables are not written while a kernel reads them: scalar loads
template <typename T>
using Constant = const __attribute__((address_space(4))) T*;
template <typename T>
__device__ __forceinline__ Constant<T> constant(const T* p) {
  return (Constant<T>)(uintptr_t)p;
}

// tile / (tiles a page), without a division: (2 tile + 1) / 2 over the tiles of a page, whose inverse in 31 bits is rounded up,
// is in the right page while tile times (tiles a page) is below 2^30 (rows_ok)
__device__ __forceinline__ int page_of(int tile, uint32_t magic) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __umulhi(2 * static_cast<uint32_t>(tile) + 1, magic);
#else
  return 0;
#endif
}

// what one workgroup does
struct RowsBlock {
  int tok0, ntok;         // tokens of its rows' list
  int block;              // which 16 RT of the list's ntok G rows
  int table;              // row of `tables`
  int kbeg, kend;         // keys
  bool whole;             // its rows have no other parts: they go to `out`
  int64_t part0;          // else row (token, head) writes part part0 + (token Hq + head) part_step
  int part_step;
  int causal0;            // >= 0: token i sees keys < causal0 + i + 1; OWN: those below its seq_lens; ALL: all (below kend, each)
};
enum : int { OWN = -1, ALL = -2 };

__device__ __forceinline__ float exp2_fast(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);
#else
  return x;
#endif
}

// joined over the four lanes that hold one row: lane ^ 16, ^ 32
template <typename F>
__device__ __forceinline__ float join_groups(float v, F f) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
#endif
  return v;
}

// Whether numbers of the wave's lanes are not all zero and all below SMALL: of bf16, which order as whole numbers do ...
struct Magnitudes {
  typedef uint16_t pair_t __attribute__((ext_vector_type(2)));
  pair_t top = {0, 0};
  __device__ __forceinline__ void take(const uint4& x, bool in) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(pair_t, in ? w[i] & 0x7FFF7FFFu : 0u));
  }
  __device__ __forceinline__ bool usual() const { return __any(max(top[0], top[1]) >= __float_as_uint(SMALL) >> 16); }
  __device__ __forceinline__ bool small() const { return !usual() && __any((top[0] | top[1]) != 0); }
};

// ... and of keys' factors (mostly the first look tells)
template <int NA>
__device__ __forceinline__ bool small_factors(const float4 (&vs)[NA]) {
  if (__any(vs[0].x >= SMALL)) return false;
  float v = 0.f;
#pragma unroll
  for (int a = 0; a < NA; ++a) v = fmaxf(fmaxf(fmaxf(v, vs[a].x), fmaxf(vs[a].y, vs[a].z)), vs[a].w);
  return !__any(v >= SMALL) && __any(v > 0.f);
}

template <int FMT, int D, int RT>
struct RowsCfg {
  static constexpr bool WIDE = FMT == KV_BF16;
  static constexpr int KK = D / 32;                  // matrix instructions over the head size
  static constexpr int MT = D / 16;                  // 16-dim tiles of the output
  static constexpr int LOADS = WIDE ? D / 32 : D / 64;   // 16-byte loads a lane, 16 tokens of K or V
  static constexpr int OROW = D + 4;                 // row of the joining buffer (padded: banks)
  static constexpr int JOIN = 4 * 16 * OROW * 4;     // bytes
  static constexpr int TURN = WIDE ? 4 * 32 * D * 2 : 0;
  static constexpr int SPACE = JOIN > TURN ? JOIN : TURN;
};

// Products q k of 32 keys -> scores less their rows' running maxima, which rise (and sums and outputs shrink) where a score is more
// than RAISE above its row's. ks, vs: the keys' and values' factors (SCALED: the keys' times softmax's scale). EDGE: some row does not
// see some key of the 32 from key0 on: its score becomes -inf. A value that is not finite then reaches the rows that see it by their
// scores, and no other by its factor (bf16: add_odd). small(): whether these keys' values (factors) are below SMALL.
template <bool EDGE, bool WIDE, bool SCALED, int NA, int RT, int MT, typename F>
__device__ __forceinline__ void scores(f32x4_t (&s)[NA][RT], const float4 (&ks)[NA], float4 (&vs)[NA], float scale, int key0, int kbeg,
                                       int kend, const int (&limit)[RT], float (&m)[RT], float (&l)[RT], float (&high)[RT],
                                       f32x4_t (&acc)[RT][MT], F small) {
  float top[RT];
  bool raise = false;
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const float f[4] = {ks[a].x, ks[a].y, ks[a].z, ks[a].w};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float k = WIDE ? scale : SCALED ? f[r] : f[r] * scale;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[a][rt][r] = fmaf(s[a][rt][r], k, -m[rt]);
    }
  }
  if constexpr (EDGE) {
    const int base = key0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      float f[4] = {vs[a].x, vs[a].y, vs[a].z, vs[a].w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = base + 16 * a + r;
        const bool odd = !WIDE && !(fabsf(f[r]) < INFINITY);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float x = odd ? NAN : s[a][rt][r];
          s[a][rt][r] = key >= kbeg && key < limit[rt] ? x : -INFINITY;
        }
        if (odd || key < kbeg || key >= kend) f[r] = 0.f;
      }
      if constexpr (!WIDE) vs[a] = make_float4(f[0], f[1], f[2], f[3]);
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = fmaxf(s[0][rt][0], s[0][rt][1]);
    top[rt] = fmaxf(fmaxf(top[rt], s[0][rt][2]), s[0][rt][3]);
#pragma unroll
    for (int a = 1; a < NA; ++a) {
      top[rt] = fmaxf(fmaxf(top[rt], s[a][rt][0]), s[a][rt][1]);
      top[rt] = fmaxf(fmaxf(top[rt], s[a][rt][2]), s[a][rt][3]);
    }
    raise = raise || top[rt] > high[rt];
  }
  if (__any(raise)) {
    bool none = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) none = none || high[rt] == -INFINITY;
    const float lift = __any(none) && small() ? LIFT_SMALL : LIFT;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const bool first = high[rt] == -INFINITY;
      float up = join_groups(top[rt], [](float x, float y) { return fmaxf(x, y); });
      if (first) {   // (maxima that would lose the lift in rounding have none: m is what the weights are relative to)
        const float on = fabsf(up) < 0x1p20f ? lift : 0.f;
        high[rt] = up == -INFINITY ? up : RAISE - on;
        up = up == -INFINITY ? 0.f : up + on;
      } else {
        up = fmaxf(up - (high[rt] - RAISE), 0.f);
      }
      const float alpha = first ? 1.f : exp2_fast(-up);
      m[rt] += up;
      l[rt] *= alpha;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][rt][r] -= up;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[rt][mt][r] *= alpha;
    }
  }
}

// ... -> weights, the P^T fragments of pairs of tiles. vs: the values' factors.
template <bool WIDE, int NA, int RT>
__device__ __forceinline__ void weights(f32x4_t (&s)[NA][RT], const float4 (&vs)[NA], float (&l)[RT], bf16x8_t (&pf)[NA / 2][RT]) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int pair = 0; pair < NA / 2; ++pair) {
      uint32_t o[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int a = 2 * pair + x;
        const float f[4] = {vs[a].x, vs[a].y, vs[a].z, vs[a].w};
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = exp2_fast(s[a][rt][r]);
          l[rt] += e[r];
          if constexpr (!WIDE) e[r] *= f[r];
        }
        o[2 * x] = pack2(e[0], e[1]);
        o[2 * x + 1] = pack2(e[2], e[3]);
      }
      pf[pair][rt] = as_frag(make_uint4(o[0], o[1], o[2], o[3]));
    }
  }
}

// bf16 pages, tiles at the edges: a value that is infinite or NaN would reach rows that do not see it, as 0 times it. Its row of V is
// zeros in the products, and is added to the rows that see it by itself.

// One load of rows of V, D / 8 lanes each, of which the caller's lanes `in` count: bits of its rows that are odd in this way, now zeros
template <int D>
__device__ __forceinline__ uint32_t odd_rows(uint4& x, bool in) {
  constexpr int LANES = D / 8;
  auto odd = [](uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; };
  const uint64_t who = __ballot(in && (odd(x.x) || odd(x.y) || odd(x.z) || odd(x.w)));
  uint32_t rows = 0;
  if (who) {
#pragma unroll
    for (int i = 0; i < 64 / LANES; ++i) rows |= (who >> (i * LANES) & ((1ull << LANES) - 1)) ? 1u << i : 0u;
    if (rows >> ((threadIdx.x & 63) / LANES) & 1) x = make_uint4(0, 0, 0, 0);
  }
  return rows;
}

// odd: such keys of the 16 NA from key0 on, s: scores, row_of: a key's row of V
template <int NA, int RT, int MT, typename F>
__device__ __forceinline__ void add_odd(uint64_t odd, const f32x4_t (&s)[NA][RT], int key0, const int (&limit)[RT], F row_of,
                                        f32x4_t (&acc)[RT][MT]) {
  const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
#pragma unroll 1
  for (; odd; odd &= odd - 1) {
    const int x = __builtin_ctzll(odd);
    const uint16_t* v = row_of(key0 + x);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float score = 0.f;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) score = x >> 4 == a && (x & 3) == r ? s[a][rt][r] : score;
      const float w = exp2_fast(__shfl(score, (x & 12) * 4 + li, 64));
      const bool seen = key0 + x < limit[rt];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint2 y = *reinterpret_cast<const uint2*>(v + 16 * mt + 4 * g);
        const float f[4] = {bf2f(y.x & 0xFFFF), bf2f(y.x >> 16), bf2f(y.y & 0xFFFF), bf2f(y.y >> 16)};
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[rt][mt][r] += seen ? w * f[r] : 0.f;
        __builtin_amdgcn_sched_barrier(0);   // (a load in flight, not all: registers)
      }
    }
  }
}

// Row r of a block's list: its fragments of Q (the dims of the K fragments), the keys it sees; `least` sinks to these.
template <int FMT, int D>
__device__ __forceinline__ void load_row(const RowsArgs& p, const RowsBlock& w, int kvh, int r, int g, bf16x8_t (&qf)[D / 32],
                                         int& limit, int& least) {
  const bool real = r < w.ntok * p.G;
  const int tok = real ? r / p.G : 0, head = kvh * p.G + (real ? r - tok * p.G : 0);
  limit = 0;
  if (real) {
    limit = w.kend;
    if (w.causal0 != ALL) {
      limit = min(limit, w.causal0 >= 0 ? w.causal0 + tok + 1 : p.seq_lens[w.tok0 + tok]);
      least = min(least, limit);
    }
  }
  const uint16_t* qp = p.q + static_cast<int64_t>(w.tok0 + tok) * p.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) {
    const int d = FMT == KV_BF16 ? 32 * kk + 8 * g : 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
    qf[kk] = as_frag(real ? ld16(qp + d) : make_uint4(0, 0, 0, 0));
  }
}

// bf16 K of 16 tokens in LDS: where 8 dims (chunk ch) of a token lie, in fragment order. The tokens of a chunk are turned by it, so
// whole rows are written and fragments read without bank conflicts. Fragments straight from the cache are 16 bytes of 16 rows, for which
// a CU's address unit takes a clock a lane in place of one for four: it was busy for 75 % of the time (64 sequences behind 4096 keys
// 39.2 -> 34.5 us, 64 heads on 8 of 20 behind 3000 21.9 -> 18.4).
template <int D>
__device__ __forceinline__ uint32_t k_chunk(int token, int ch) {
  return ((ch * 16) + (token ^ (ch & 7))) * 16;
}

template <int FMT, int D, int RT, bool ONCE>
__device__ __forceinline__ void attend_rows(const RowsArgs& p, const RowsBlock w, int kvh, uint8_t* space,
                                            float (*m_lds)[16 * RT], float (*l_lds)[16 * RT]) {
  using C = RowsCfg<FMT, D, RT>;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15;
  const int nrows = w.ntok * p.G, row0 = w.block * 16 * RT;

  float m[RT], l[RT], high[RT];   // running maximum and sum; what a score has to pass to raise it: anything, before the first key
  f32x4_t acc[RT][C::MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = l[rt] = 0.f;
    high[rt] = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt) acc[rt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int tpp = p.bs >> 4;                       // tiles a page
  const int t_end = (w.kend + 31) >> 5, last = max((w.kend + 15) / 16 - 1, 0);
  const Constant<int32_t> table = constant(p.tables + w.table * p.table_stride);
  uint4 kr[2][C::LOADS], vr[2][C::LOADS];
  float4 ks[2], vs[2];
  // a decode step reads its 8-bit keys once (non-temporal); blocks of rows over the same keys find them in the L2. (bf16: 64 sequences
  // behind 4096 keys 34.5 us, with their own keys non-temporal 38.6)
  auto load16 = [](const void* at) { return ONCE && !C::WIDE ? ld16_nt(at) : ld16(at); };
  // where the halves of a tile lie: clamped to the last tile that holds a key, and into the cache. The page numbers of the
  // tile after the next are asked for while the next one's loads go out, so no load waits for its address. Addresses are scalar
  // work of each tile (a third of the loop's instructions where they came from the indexes each time): one offset for K and V
  const uint32_t elem = C::WIDE ? 2 : 1;
  const uint32_t page_bytes = static_cast<uint32_t>(p.Hkv) * p.bs * D * elem, page_scales = static_cast<uint32_t>(p.Hkv) * 2 * p.bs;
  const uint8_t* k_head = p.k + static_cast<int64_t>(kvh) * p.bs * D * elem;
  const uint8_t* v_head = p.v + static_cast<int64_t>(kvh) * p.bs * D * elem;
  const float* s_head = p.scales + static_cast<int64_t>(kvh) * 2 * p.bs;
  int page[2], off[2];
  auto find = [&](int t) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int tile = min(2 * t + a, last), pg = page_of(tile, p.page_magic);
      page[a] = table[pg];
      off[a] = (tile - pg * tpp) * 16;
    }
  };
  uint64_t at[2];                // bytes of the half's tile from k_head, v_head
  const float* factor[2];        // its first scale
  auto settle = [&]() {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint32_t pg = min(max(page[a], 0), p.num_blocks - 1);
      at[a] = static_cast<uint64_t>(pg) * page_bytes + static_cast<uint32_t>(off[a]) * D * elem;
      if constexpr (!C::WIDE) factor[a] = s_head + static_cast<uint64_t>(pg) * page_scales + static_cast<uint32_t>(off[a]);
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint8_t* base = k_head + at[a];
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) kr[a][i] = load16(base + static_cast<uint32_t>(lane * 16 + 1024 * i));
      if constexpr (!C::WIDE) ks[a] = *reinterpret_cast<const float4*>(factor[a] + 4 * g);
    }
  };
  auto load_v = [&]() {          // (bf16: 4 (D 128) or 8 whole rows a load)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint8_t* base = v_head + at[a];
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) vr[a][i] = load16(base + static_cast<uint32_t>(lane * 16 + 1024 * i));
      if constexpr (!C::WIDE) vs[a] = *reinterpret_cast<const float4*>(factor[a] + p.bs + 4 * g);
    }
  };
  // The wave's tiles t0 + 4 i, in an order that leaves those at the edges (some row does not see some key) to a loop of their own:
  // what they ask for would be selects in every tile's way, and two bodies in one loop copy the sums from one to the other
  const int t0 = (w.kbeg >> 5) + wid, n = t0 < t_end ? (t_end - t0 + 3) >> 2 : 0;
  const int ahead = n > 0 && 32 * t0 < w.kbeg ? 1 : 0;                         // the first tile is one: it goes last
  auto nth = [&](int j) {                                                      // (behind the last: anything)
    const int i = j + ahead;
    return t0 + 4 * (i < n ? i : 0);
  };
  if (n > 0) {
    find(nth(0));
    settle();
    load_k();
    load_v();
    find(nth(1));
  }
  // rows: fragments of Q, and the keys that each sees (asked for after the first keys, which come from further away)
  int limit[RT];
  int least = w.kend;   // every row sees the keys below
  bf16x8_t qf[RT][C::KK];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) load_row<FMT, D>(p, w, kvh, row0 + rt * 16 + li, g, qf[rt], limit[rt], least);
  if (w.causal0 != ALL)
    for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
  least = __builtin_amdgcn_readfirstlane(least);
  // no row sees the keys from here on, which may never have been written
  int end = w.kend;
  if (w.causal0 == OWN) {
    int most = limit[0];
#pragma unroll
    for (int rt = 1; rt < RT; ++rt) most = max(most, limit[rt]);
    for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor(most, o, 64));
    end = __builtin_amdgcn_readfirstlane(most);
  }
  const int whole = max(0, min(n, ((least >> 5) - t0 + 3) >> 2) - ahead);      // tiles that every row sees
  // S^T of the tile whose K is in registers
  auto product = [&](f32x4_t (&s)[2][RT]) {
    uint8_t* turn = space + wid * 64 * D;
    if constexpr (C::WIDE) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) st16(turn + a * 32 * D + k_chunk<D>((lane + 64 * i) / (D / 8), (lane + 64 * i) % (D / 8)), kr[a][i]);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[a][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) {
#pragma unroll
        for (int x = 0; x < (C::WIDE ? 1 : 2); ++x) {
          const int kk = C::WIDE ? i : 2 * i + x;
          bf16x8_t kx;
          if constexpr (C::WIDE) kx = as_frag(ld16(turn + a * 32 * D + k_chunk<D>(li, 4 * i + g)));
          else kx = x == 0 ? kv_widen8<FMT>(kr[a][i].x, kr[a][i].y) : kv_widen8<FMT>(kr[a][i].z, kr[a][i].w);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[a][rt] = mfma16x16x32(kx, qf[rt][kk], s[a][rt]);
        }
      }
    }
  };
  auto row_of = [&](int key) {   // of V
    const int pg = page_of(key >> 4, p.page_magic);
    return reinterpret_cast<const uint16_t*>(v_head + static_cast<uint64_t>(min(max(table[pg], 0), p.num_blocks - 1)) * page_bytes) +
           (key - pg * p.bs) * D;
  };
  // scores of tile t, whose V is in registers; bf16: its odd rows
  auto judge = [&](int t, f32x4_t (&s)[2][RT], const float4 (&factors)[2], auto edge) {
    uint32_t odd = 0;
    auto small = [&]() {
      if constexpr (C::WIDE) {
        Magnitudes x;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int i = 0; i < C::LOADS; ++i) {
            const int key = 32 * t + 16 * a + (lane + 64 * i) / (D / 8);
            x.take(vr[a][i], key >= w.kbeg && key < end);
            if (a == 0 && i == 0 && x.usual()) return false;
          }
        return x.small();
      } else {
        return small_factors(vs);
      }
    };
    scores<decltype(edge)::value, C::WIDE, false, 2, RT, C::MT>(s, factors, vs, p.scale, 32 * t, w.kbeg, end, limit, m, l, high, acc, small);
    if constexpr (decltype(edge)::value) {   // V of keys outside the range: anything (E4M3's NaN too), so zeros
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        if constexpr (C::WIDE) {
#pragma unroll
          for (int i = 0; i < C::LOADS; ++i) {
            const int key = 32 * t + 16 * a + (lane + 64 * i) / (D / 8);
            const bool in = key >= w.kbeg && key < end;
            if (!in) vr[a][i] = make_uint4(0, 0, 0, 0);
            if constexpr (!ONCE) odd |= odd_rows<D>(vr[a][i], in) << (16 * a + 64 / (D / 8) * i);   // (once: all rows see the same keys)
          }
        } else {
          uint32_t keep = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = 32 * t + 16 * a + 4 * g + r;
            keep |= key >= w.kbeg && key < end ? 0xFFu << (8 * r) : 0u;
          }
#pragma unroll
          for (int i = 0; i < C::LOADS; ++i) vr[a][i] = make_uint4(vr[a][i].x & keep, vr[a][i].y & keep, vr[a][i].z & keep, vr[a][i].w & keep);
        }
      }
    }
    return odd;
  };
  auto step = [&](int j, auto edge) {
    f32x4_t s[2][RT];
    product(s);
    const float4 factors[2] = {ks[0], ks[1]};
    settle();
    load_k();
    const uint32_t odd = judge(nth(j), s, factors, edge);
    bf16x8_t pf[1][RT];
    weights<C::WIDE, 2, RT>(s, vs, l, pf);
    if constexpr (C::WIDE && !ONCE && decltype(edge)::value) {
      if (odd) add_odd(odd, s, 32 * nth(j), limit, row_of, acc);
    }
    uint16_t* turn = reinterpret_cast<uint16_t*>(space) + wid * 32 * D;
    if constexpr (C::WIDE) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) {
          const int row = 16 * a + (lane + 64 * i) / (D / 8), ch = (lane + 64 * i) % (D / 8);
          st16(turn + row * D + (ch ^ (((row & 7) << 1) & (D / 8 - 1))) * 8, vr[a][i]);
        }
      load_v();
    }
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt) {
      bf16x8_t vx;
      if constexpr (C::WIDE) {
        const int row = 4 * g + (li >> 2), col = mt * 16 + 4 * (li & 3);
        const uint16_t* src = turn + row * D + ((col >> 3) ^ (((row & 7) << 1) & (D / 8 - 1))) * 8 + (col & 7);
        const uint2 lo = __builtin_bit_cast(uint2, lds_read_tr16(src)), hi = __builtin_bit_cast(uint2, lds_read_tr16(src + 16 * D));
        vx = as_frag(make_uint4(lo.x, lo.y, hi.x, hi.y));
      } else {
        const uint4 &va = vr[0][mt >> 2], &vb = vr[1][mt >> 2];
        vx = kv_widen8<FMT>((mt & 3) == 0 ? va.x : (mt & 3) == 1 ? va.y : (mt & 3) == 2 ? va.z : va.w,
                            (mt & 3) == 0 ? vb.x : (mt & 3) == 1 ? vb.y : (mt & 3) == 2 ? vb.z : vb.w);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt][mt] = mfma16x16x32(vx, pf[0][rt], acc[rt][mt]);
    }
    if constexpr (!C::WIDE) load_v();
    find(nth(j + 2));
  };
#pragma unroll 1
  for (int j = 0; j < whole; ++j) step(j, std::false_type{});
#pragma unroll 1
  for (int j = whole; j < n; ++j) step(j, std::true_type{});

  // ---- the four waves' states: O^T[16 mt + 4 g + r][row li] of each row tile
  float* o_lds = reinterpret_cast<float*>(space);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = join_groups(l[rt], [](float x, float y) { return x + y; });
    if (g == 0) {
      m_lds[wid][rt * 16 + li] = sum == 0.f ? LOWEST : m[rt];
      l_lds[wid][rt * 16 + li] = sum;
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    __syncthreads();   // (the rows' last reads of this buffer)
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt)
      *reinterpret_cast<float4*>(o_lds + (wid * 16 + li) * C::OROW + mt * 16 + 4 * g) =
          make_float4(acc[rt][mt][0], acc[rt][mt][1], acc[rt][mt][2], acc[rt][mt][3]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * D / 4; idx += 256) {
      const int i = idx / (D / 4), d = idx % (D / 4) * 4, r = row0 + rt * 16 + i;
      if (r >= nrows) continue;
      float M = LOWEST;
#pragma unroll
      for (int x = 0; x < 4; ++x) M = fmaxf(M, m_lds[x][rt * 16 + i]);
      float sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float e = exp2_fast(m_lds[x][rt * 16 + i] - M);
        const float4 a = *reinterpret_cast<const float4*>(o_lds + (x * 16 + i) * C::OROW + d);
        sum += l_lds[x][rt * 16 + i] * e;
        o.x += a.x * e; o.y += a.y * e; o.z += a.z * e; o.w += a.w * e;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;   // (a row that sees no key)
      const int tok = r / p.G, head = kvh * p.G + r - tok * p.G;
      const int64_t at = static_cast<int64_t>(w.tok0 + tok);
      if (w.whole) {
        *reinterpret_cast<uint2*>(p.out + at * p.out_stride + static_cast<int64_t>(head) * D + d) =
            make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
      } else {
        const int64_t part = w.part0 + (at * p.Hq + head) * w.part_step;
        *reinterpret_cast<float4*>(p.part_out + part * D + d) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (d == 0) p.part_lse[part] = sum == 0.f ? -INFINITY : M + __log2f(sum);
      }
    }
  }
}

// ---- many rows: 128 a workgroup, 32 a wave, all over the same keys ------------------------------------------------------
// The widening of 8-bit codes is vector work, and that (with the softmax) bounds blocks of many rows, not the products: here a
// stage of 64 keys is widened once for the workgroup's 128 rows and laid in LDS in fragment order, two stages in turn, one
// barrier a stage. Each wave has rows of its own, so nothing is joined at the end. Ranges begin at multiples of 32 keys.
template <int FMT, int D>
struct BlockCfg {
  static constexpr bool WIDE = FMT == KV_BF16;
  static constexpr int ROWS = 128, KEYS = 64, RT = 2;
  static constexpr int KK = D / 32, MT = D / 16;
  static constexpr int SIDE = KEYS * D * 2;               // bytes of a stage's K, or V
  static constexpr int STAGE = 2 * SIDE + 2 * KEYS * 4;   // and the scales
  static constexpr int SPACE = 2 * STAGE;
  static constexpr int RAW = WIDE ? D / 32 : D / 64;      // 16-byte loads a lane for its 16 keys of K, and as many of V
};

template <int FMT, int D>
__device__ __forceinline__ void attend_block(const RowsArgs& p, const RowsBlock w, int kvh, uint8_t* space) {
  using C = BlockCfg<FMT, D>;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15;
  const int row0 = w.block * C::ROWS + wid * 32;
  int limit[C::RT], least = w.kend;
  bf16x8_t qf[C::RT][C::KK];
#pragma unroll
  for (int rt = 0; rt < C::RT; ++rt) load_row<FMT, D>(p, w, kvh, row0 + rt * 16 + li, g, qf[rt], limit[rt], least);
  int most = max(limit[0], limit[1]);
  for (int o = 1; o < 16; o <<= 1) {
    least = min(least, __shfl_xor(least, o, 64));
    most = max(most, __shfl_xor(most, o, 64));
  }
  most = __builtin_amdgcn_readfirstlane(most);   // no row of the wave sees the keys from here on
  int* of_waves = reinterpret_cast<int*>(space);
  if (lane == 0) {
    of_waves[wid] = least;
    of_waves[4 + wid] = most;
  }
  __syncthreads();
  least = __builtin_amdgcn_readfirstlane(min(min(of_waves[0], of_waves[1]), min(of_waves[2], of_waves[3])));
  const int kend = __builtin_amdgcn_readfirstlane(max(max(of_waves[4], of_waves[5]), max(of_waves[6], of_waves[7])));   // and none of these
  __syncthreads();

  float m[C::RT], l[C::RT], high[C::RT];
  f32x4_t acc[C::RT][C::MT];
#pragma unroll
  for (int rt = 0; rt < C::RT; ++rt) {
    m[rt] = l[rt] = 0.f;
    high[rt] = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt) acc[rt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int tpp = p.bs >> 4, last = max((kend + 15) / 16 - 1, 0);
  const int stages = kend > w.kbeg ? (kend - w.kbeg + C::KEYS - 1) / C::KEYS : 0;
  const Constant<int32_t> table = constant(p.tables + w.table * p.table_stride);
  const uint32_t elem = C::WIDE ? 2 : 1;
  const uint32_t page_bytes = static_cast<uint32_t>(p.Hkv) * p.bs * D * elem, page_scales = static_cast<uint32_t>(p.Hkv) * 2 * p.bs;
  const uint8_t* k_head = p.k + static_cast<int64_t>(kvh) * p.bs * D * elem;
  const uint8_t* v_head = p.v + static_cast<int64_t>(kvh) * p.bs * D * elem;
  const float* s_head = p.scales + static_cast<int64_t>(kvh) * 2 * p.bs;
  // Of a stage's four tiles, wave w brings K (and the scales) of tile w; of V, 8-bit codes of 128 dims: half w & 1 of the dims of both
  // tiles of pair w >> 1, which a fragment has side by side; else tile w. Page numbers are asked for a stage ahead of the loads.
  constexpr bool PAIRED = !C::WIDE && D == 128;
  int page[2], off[2];
  auto find = [&](int stage) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int tile = min((w.kbeg >> 4) + 4 * stage + (wid & 2) + a, last), pg = page_of(tile, p.page_magic);
      page[a] = table[pg];
      off[a] = (tile - pg * tpp) * 16;
    }
  };
  uint4 kraw[C::RAW], vraw[C::RAW];
  float factor = 0.f;
  auto fetch = [&]() {
    uint64_t at[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      page[a] = min(max(page[a], 0), p.num_blocks - 1);
      at[a] = static_cast<uint64_t>(static_cast<uint32_t>(page[a])) * page_bytes + static_cast<uint32_t>(off[a]) * D * elem;
    }
    const int own = wid & 1;
    const uint8_t* kb = k_head + (own ? at[1] : at[0]);
#pragma unroll
    for (int i = 0; i < C::RAW; ++i)
      kraw[i] = ld16(kb + (C::WIDE ? static_cast<uint32_t>(li * D * 2 + 16 * g + 64 * i) : static_cast<uint32_t>(lane * 16 + 1024 * i)));
    if constexpr (PAIRED) {
#pragma unroll
      for (int a = 0; a < 2; ++a) vraw[a] = ld16(v_head + at[a] + static_cast<uint32_t>(own * 1024 + lane * 16));
    } else {
      const uint8_t* vb = v_head + (own ? at[1] : at[0]);
#pragma unroll
      for (int i = 0; i < C::RAW; ++i) vraw[i] = ld16(vb + static_cast<uint32_t>(lane * 16 + 1024 * i));
    }
    if constexpr (!C::WIDE) {   // lanes 0 .. 15: the keys', 16 .. 31: the values'
      const float* sc = s_head + static_cast<uint64_t>(static_cast<uint32_t>(own ? page[1] : page[0])) * page_scales +
                        static_cast<uint32_t>(own ? off[1] : off[0]);
      factor = sc[static_cast<uint32_t>((g & 1) * p.bs + li)];
    }
  };
  auto row_of = [&](int key) {   // of V
    const int pg = page_of(key >> 4, p.page_magic);
    return reinterpret_cast<const uint16_t*>(v_head + static_cast<uint64_t>(min(max(table[pg], 0), p.num_blocks - 1)) * page_bytes) +
           (key - pg * p.bs) * D;
  };
  auto kept = [&](int key) { return key >= w.kbeg && key < kend; };
  auto lay = [&](int stage, auto edge) {
    uint8_t* kd = space + (stage & 1) * C::STAGE;
    uint8_t* vd = kd + C::SIDE;
    const int key0 = w.kbeg + stage * C::KEYS;
    if constexpr (C::WIDE) {
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < C::RAW; ++i) {
        st16(kd + ((wid * C::KK + i) * 64 + lane) * 16, kraw[i]);
        const int row = 16 * wid + (lane + 64 * i) / (D / 8), ch = (lane + 64 * i) % (D / 8);
        uint4 x = vraw[i];
        if constexpr (decltype(edge)::value) {
          const bool in = kept(key0 + row);
          if (!in) x = make_uint4(0, 0, 0, 0);
          odd |= odd_rows<D>(x, in) << (64 / (D / 8) * i);
        }
        st16(vd + (row * (D / 8) + (ch ^ (((row & 7) << 1) & (D / 8 - 1)))) * 16, x);
      }
      if (lane == 0) reinterpret_cast<uint16_t*>(kd + 2 * C::SIDE)[wid] = odd;
    } else {
#pragma unroll
      for (int i = 0; i < C::RAW; ++i) {
        st16(kd + ((wid * C::KK + 2 * i) * 64 + lane) * 16, __builtin_bit_cast(uint4, kv_widen8<FMT>(kraw[i].x, kraw[i].y)));
        st16(kd + ((wid * C::KK + 2 * i + 1) * 64 + lane) * 16, __builtin_bit_cast(uint4, kv_widen8<FMT>(kraw[i].z, kraw[i].w)));
      }
      if constexpr (decltype(edge)::value) {   // V of keys outside the range may be anything (E4M3's NaN too): zeros
#pragma unroll
        for (int a = 0; a < C::RAW; ++a) {
          const int tile = PAIRED ? (wid & 2) + a : wid;
          uint32_t keep = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) keep |= kept(key0 + 16 * tile + 4 * g + r) ? 0xFFu << (8 * r) : 0u;
          vraw[a] = make_uint4(vraw[a].x & keep, vraw[a].y & keep, vraw[a].z & keep, vraw[a].w & keep);
        }
      }
      if constexpr (PAIRED) {
        const uint32_t x[4] = {vraw[0].x, vraw[0].y, vraw[0].z, vraw[0].w}, y[4] = {vraw[1].x, vraw[1].y, vraw[1].z, vraw[1].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st16(vd + (((wid >> 1) * C::MT + (wid & 1) * 4 + i) * 64 + lane) * 16, __builtin_bit_cast(uint4, kv_widen8<FMT>(x[i], y[i])));
      } else {
        const uint32_t x[4] = {vraw[0].x, vraw[0].y, vraw[0].z, vraw[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint2*>(vd + (((wid >> 1) * C::MT + i) * 64 + lane) * 16 + (wid & 1) * 8) = kv_widen4<FMT>(x[i]);
      }
      if (lane < 32) reinterpret_cast<float*>(kd + 2 * C::SIDE)[g * C::KEYS + wid * 16 + li] = g ? factor : factor * p.scale;
    }
  };
  if (stages > 0) {
    find(0);
    fetch();
    find(1);   // (stages behind the last: clamped to its last tile, and unused)
    lay(0, std::true_type{});
    fetch();
    find(2);
  }
  __syncthreads();
  auto step = [&](int stage, auto edge) {
    lay(stage + 1, edge);
    fetch();
    find(stage + 3);
    const uint8_t* kd = space + (stage & 1) * C::STAGE;
    const uint8_t* vd = kd + C::SIDE;
    const float* sd = reinterpret_cast<const float*>(kd + 2 * C::SIDE) + 4 * g;
    const int key0 = w.kbeg + stage * C::KEYS;
    if (!decltype(edge)::value || key0 < most) {
      f32x4_t s[4][C::RT];
      float4 ks[4], vs[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
#pragma unroll
        for (int rt = 0; rt < C::RT; ++rt) s[a][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < C::KK; ++kk) {
          const bf16x8_t kx = as_frag(ld16(kd + ((a * C::KK + kk) * 64 + lane) * 16));
#pragma unroll
          for (int rt = 0; rt < C::RT; ++rt) s[a][rt] = mfma16x16x32(kx, qf[rt][kk], s[a][rt]);
        }
        if constexpr (!C::WIDE) {
          ks[a] = *reinterpret_cast<const float4*>(sd + 16 * a);
          vs[a] = *reinterpret_cast<const float4*>(sd + C::KEYS + 16 * a);
        }
      }
      auto small = [&]() {
        if constexpr (C::WIDE) {
          Magnitudes x;
#pragma unroll
          for (int i = 0; i < C::SIDE / 1024; ++i) {   // (zeros outside the range)
            x.take(ld16(vd + (lane + 64 * i) * 16), true);
            if (i == 0 && x.usual()) return false;
          }
          return x.small();
        } else {
          return small_factors(vs);
        }
      };
      scores<decltype(edge)::value, C::WIDE, true, 4, C::RT, C::MT>(s, ks, vs, p.scale, key0, w.kbeg, kend, limit, m, l, high, acc, small);
      bf16x8_t pf[2][C::RT];
      weights<C::WIDE, 4, C::RT>(s, vs, l, pf);
      if constexpr (C::WIDE && decltype(edge)::value) {
        const uint2 o = *reinterpret_cast<const uint2*>(kd + 2 * C::SIDE);
        const uint64_t odd = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(o.y)) << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(o.x));
        if (odd) add_odd(odd, s, key0, limit, row_of, acc);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
          bf16x8_t vx;
          if constexpr (C::WIDE) {
            const int row = 32 * half + 4 * g + (li >> 2), col = mt * 16 + 4 * (li & 3);
            const uint16_t* src = reinterpret_cast<const uint16_t*>(vd) + row * D +
                                  ((col >> 3) ^ (((row & 7) << 1) & (D / 8 - 1))) * 8 + (col & 7);
            const uint2 lo = __builtin_bit_cast(uint2, lds_read_tr16(src)), hi = __builtin_bit_cast(uint2, lds_read_tr16(src + 16 * D));
            vx = as_frag(make_uint4(lo.x, lo.y, hi.x, hi.y));
          } else {
            vx = as_frag(ld16(vd + ((half * C::MT + mt) * 64 + lane) * 16));
          }
#pragma unroll
          for (int rt = 0; rt < C::RT; ++rt) acc[rt][mt] = mfma16x16x32(vx, pf[half][rt], acc[rt][mt]);
        }
    }
    __syncthreads();
  };
  // stages that every row sees (and whose next one, laid down meanwhile, ends within the range, and of bf16 is seen by every row too),
  // then the others: two loops, as above
  const int whole = max(0, min(min((least - w.kbeg) / C::KEYS - (C::WIDE ? 1 : 0), stages), (kend - w.kbeg) / C::KEYS - 1));
#pragma unroll 1
  for (int stage = 0; stage < whole; ++stage) step(stage, std::false_type{});
#pragma unroll 1
  for (int stage = whole; stage < stages; ++stage) step(stage, std::true_type{});

#pragma unroll
  for (int rt = 0; rt < C::RT; ++rt) {
    const int r = row0 + rt * 16 + li;
    const float sum = join_groups(l[rt], [](float x, float y) { return x + y; });
    if (r >= w.ntok * p.G) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tok = r / p.G, head = kvh * p.G + r - tok * p.G;
    const int64_t at = static_cast<int64_t>(w.tok0 + tok);
    if (w.whole) {
      uint16_t* dst = p.out + at * p.out_stride + static_cast<int64_t>(head) * D + 4 * g;
#pragma unroll
      for (int mt = 0; mt < C::MT; ++mt)
        *reinterpret_cast<uint2*>(dst + 16 * mt) = make_uint2(pack2(acc[rt][mt][0] * inv, acc[rt][mt][1] * inv),
                                                              pack2(acc[rt][mt][2] * inv, acc[rt][mt][3] * inv));
    } else {
      const int64_t part = w.part0 + (at * p.Hq + head) * w.part_step;
#pragma unroll
      for (int mt = 0; mt < C::MT; ++mt)
        *reinterpret_cast<float4*>(p.part_out + part * D + 16 * mt + 4 * g) =
            make_float4(acc[rt][mt][0] * inv, acc[rt][mt][1] * inv, acc[rt][mt][2] * inv, acc[rt][mt][3] * inv);
      if (g == 0) p.part_lse[part] = sum == 0.f ? -INFINITY : m[rt] + __log2f(sum);
    }
  }
}

#define XGK_ROWS_LDS(FMT, D, RT)                                                                         \
  __shared__ __attribute__((aligned(16))) uint8_t space[RowsCfg<FMT, D, RT>::SPACE];                    \
  __shared__ float m_lds[4][16 * RT], l_lds[4][16 * RT]

// share `split` of `splits` of the 32-key tiles of [kbeg, kend)
__device__ __forceinline__ void share(int& kbeg, int& kend, int split, int splits) {
  if (splits <= 1) return;
  const int first = kbeg >> 5, tiles = max(0, ((kend + 31) >> 5) - first), each = (tiles + splits - 1) / splits;
  kbeg = max(kbeg, 32 * (first + split * each));
  kend = min(kend, 32 * (first + min(tiles, (split + 1) * each)));
}

// ---- decode: shares of the batch's keys -------------------------------------------------------------------------------------
// A batch's sequences are of any lengths, which the host does not know, so the keys are shared out here: of `shares` workgroups a kv
// head (and block of 16 query heads) each takes up to `run` units of 128 keys (a 32-key tile a wave) of one sequence, with run the
// batch's units over shares - B, and `least` where none has more: a short search, for share i is sequence i then (256 sequences of
// 300 - 900 keys 71 -> 68 us). So a sequence has ceil(units / run) parts, at least one and MAX_PARTS at most (the join's factors leave
// room for 256 with those of the common keys), and all have shares at most. (With as many parts for each sequence the longest one
// bounds the step: 1 sequence of 60 k keys beside 63 of 500, fp8, takes 428 us whole and 41 so.) The limit leaves CUs idle where few
// long sequences have one kv head: 1 of 131072 keys, 8 / 1 heads of 128, fp8, 17.7 us for a floor of 7.3, 2 20.4 for 14.5.
constexpr int MAX_PARTS = 128;

template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
#if defined(__HIP_DEVICE_COMPILE__)
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
#else
  return v;
#endif
}
// sums of the lanes up to each
__device__ __forceinline__ int wave_scan(int v) {
  v = scan_step<0x111, 0xF>(v);
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);
  return scan_step<0x143, 0xC>(v);
}

struct Share {
  int b, part;            // sequence (-1: none) and which of its parts
  int parts, first;       // its parts, and the share that is its first
  int kbeg, kend;
};

__device__ __forceinline__ void own_keys(const RowsArgs& p, const int32_t* starts, int b, int& kbeg, int& kend) {
  kend = min(max(p.seq_lens[b], 0), p.width * p.bs);
  kbeg = starts ? min(max(starts[b], 0), kend) : 0;
}

// Share i, or (of >= 0) the first share of sequence `of`, of a batch whose keys are cut; AT_ONCE lengths a lane at a time.
template <int AT_ONCE>
__device__ __forceinline__ void cut_share(const RowsArgs& p, const int32_t* starts, int B, int shares, int i, int of, Share& s, int& run) {
  const int lane = threadIdx.x & 63;
  int u[AT_ONCE];
  auto units = [&](int b0) {
    int kbeg[AT_ONCE], kend[AT_ONCE];
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a) own_keys(p, starts, min(b0 + 64 * a + lane, B - 1), kbeg[a], kend[a]);
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a)
      u[a] = b0 + 64 * a + lane < B && kend[a] > kbeg[a] ? (((kend[a] + 31) >> 5) - (kbeg[a] >> 5) + 3) >> 2 : 0;
  };
  bool cut = false;
  for (int b0 = 0; b0 < B; b0 += 64 * AT_ONCE) {
    units(b0);
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a) cut = cut || __any(u[a] > p.least);
  }
  if (!cut) {   // one part each
    const int b = of >= 0 ? of : i;
    s.b = b < B ? b : -1;
    s.first = b;
    return;
  }
  int all = 0, most = 0;
  for (int b0 = 0; b0 < B; b0 += 64 * AT_ONCE) {
    if (B > 64 * AT_ONCE) units(b0);
    int sum = 0;
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a) {
      sum += u[a];
      most = max(most, u[a]);
    }
    all += __builtin_amdgcn_readlane(wave_scan(sum), 63);
  }
  most = __float_as_int(wave_join(__int_as_float(most), [](float x, float y) { return __int_as_float(max(__float_as_int(x), __float_as_int(y))); }));
  run = __builtin_amdgcn_readfirstlane(max(max(p.least, (all + shares - B - 1) / (shares - B)), (most + MAX_PARTS - 1) / MAX_PARTS));
  int before = 0;
  for (int b0 = 0; b0 < B && s.b < 0; b0 += 64 * AT_ONCE) {
    if (B > 64 * AT_ONCE) units(b0);
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a) {
      const int b = b0 + 64 * a + lane, parts = b < B ? max(1, (u[a] + run - 1) / run) : 0;
      const int upto = before + wave_scan(parts);
      const uint64_t who = __ballot(of >= 0 ? b == of : i >= upto - parts && i < upto);
      if (who) {
        const int l = __builtin_ctzll(who);
        s.b = b0 + 64 * a + l;
        s.parts = __builtin_amdgcn_readlane(parts, l);
        s.first = __builtin_amdgcn_readlane(upto, l) - s.parts;
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
  }
}

// All lanes of the wave take part.
__device__ __forceinline__ Share find_share(const RowsArgs& p, const int32_t* starts, int B, int shares, int i, int of) {
  Share s{-1, 0, 1, 0, 0, 0};
  int run = 0;
  if (shares <= B) {
    s.b = s.first = of >= 0 ? of : i;
    if (s.b >= B) s.b = -1;
  } else if (B <= 64) {
    cut_share<1>(p, starts, B, shares, i, of, s, run);
  } else {
    cut_share<4>(p, starts, B, shares, i, of, s, run);
  }
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.first = __builtin_amdgcn_readfirstlane(s.first);
  s.parts = __builtin_amdgcn_readfirstlane(s.parts);
  s.part = of >= 0 ? 0 : i - s.first;
  if (s.b >= 0) {
    own_keys(p, starts, s.b, s.kbeg, s.kend);
    s.kbeg = __builtin_amdgcn_readfirstlane(s.kbeg);
    s.kend = __builtin_amdgcn_readfirstlane(s.kend);
    if (s.parts > 1) {
      const int first = s.kbeg >> 5;
      s.kend = min(s.kend, 32 * (first + (s.part + 1) * 4 * run));
      s.kbeg = max(s.kbeg, 32 * (first + s.part * 4 * run));
    }
  }
  return s;
}

// Share i of the sequences' new tokens, block `block` of their heads. counts: each sequence's parts besides.
template <int FMT, int D>
__device__ __forceinline__ void decode_share(const RowsArgs& p, int kvh, const int32_t* starts, const int32_t* counts, int B, int shares,
                                             int i, int block, int64_t part0, uint8_t* space, float (*m_lds)[16], float (*l_lds)[16]) {
  const Share s = find_share(p, starts, B, shares, i, -1);
  if (s.b < 0) return;
  RowsBlock w;
  w.tok0 = w.table = s.b;
  w.ntok = 1;
  w.block = block;
  w.kbeg = s.kbeg;
  w.kend = s.kend;
  if (w.kbeg >= w.kend) w.kbeg = w.kend = 0;
  w.whole = s.parts == 1 && !(counts && counts[s.b] > 0);
  w.part0 = part0 + static_cast<int64_t>(i - s.b) * p.Hq;   // (share i's rows: i Hq + head)
  w.part_step = 1;
  w.causal0 = ALL;
  attend_rows<FMT, D, 1, true>(p, w, kvh, space, m_lds, l_lds);
}

// One new token of each sequence. Grid (Hkv, shares heads' blocks of 16).
template <int FMT, int D>
__global__ void __launch_bounds__(256, 3) rows_decode_kernel(RowsArgs p, int B, int blocks, int shares) {
  XGK_ROWS_LDS(FMT, D, 1);
  const int i = blockIdx.y / blocks;
  decode_share<FMT, D>(p, blockIdx.x, nullptr, nullptr, B, shares, i, blockIdx.y - i * blocks, 0, space, m_lds, l_lds);
}

// Prompt portions, causal. Grid (Hkv, blocks of rows of the longest, sequences splits). Late blocks see the most keys: first.
template <int FMT, int D, int RT>
__global__ void __launch_bounds__(256, RT <= 1 || D == 64 ? 3 : 2) rows_prompt_kernel(RowsArgs p, const int32_t* qsl, int tokens, int splits) {
  const int s = blockIdx.z / splits;
  RowsBlock w;
  w.tok0 = min(max(qsl[s], 0), tokens);
  w.ntok = min(max(qsl[s + 1], 0), tokens) - w.tok0;
  w.block = gridDim.y - 1 - blockIdx.y;
  if (w.ntok <= 0 || w.block * 16 * RT >= w.ntok * p.G) return;
  w.table = s;
  const int len = min(p.seq_lens[s], p.width * p.bs);
  w.causal0 = max(p.seq_lens[s] - w.ntok, 0);   // tokens before the portion
  const int last_tok = min(w.ntok - 1, ((w.block + 1) * 16 * RT - 1) / p.G);
  w.kbeg = 0;
  w.kend = max(0, min(len, w.causal0 + last_tok + 1));
  share(w.kbeg, w.kend, blockIdx.z - s * splits, splits);
  if (w.kbeg >= w.kend) w.kbeg = w.kend = 0;
  w.whole = splits == 1;
  w.part0 = blockIdx.z - s * splits;
  w.part_step = splits;
  if constexpr (RT == 8) {
    __shared__ __attribute__((aligned(16))) uint8_t space[BlockCfg<FMT, D>::SPACE];
    attend_block<FMT, D>(p, w, blockIdx.x, space);
  } else {
    XGK_ROWS_LDS(FMT, D, RT);
    attend_rows<FMT, D, RT, false>(p, w, blockIdx.x, space, m_lds, l_lds);
  }
}

// Groups of decode rows with common keys, in one launch: first the common parts (items [n][8]: first sequence, sequences, block of
// rows, first key, end key, slot), then the shares of the sequences' own keys. The first are bound by the vector and matrix work, the
// others by HBM, and run beside each other. Grid (Hkv, n_items + shares heads' blocks of 16). Parts: slots a row of the common
// ones, then the shares'.
template <int FMT, int D, int RT>
__global__ void __launch_bounds__(256, RT == 1 && !(FMT == KV_BF16 && D == 128) ? 3 : 2) rows_shared_kernel(RowsArgs p, const int32_t* items, int n_items, const int32_t* prefix,
                                                             const int32_t* counts, int slots, int B, int blocks, int shares) {
  constexpr int SPACE = RT == 8 && BlockCfg<FMT, D>::SPACE > RowsCfg<FMT, D, 2>::SPACE ? BlockCfg<FMT, D>::SPACE : RowsCfg<FMT, D, 2>::SPACE;
  constexpr int LISTS = RT == 8 ? 1 : RT;
  __shared__ __attribute__((aligned(16))) uint8_t space[SPACE];
  __shared__ float m_lds[4][16 * LISTS], l_lds[4][16 * LISTS];
  if (blockIdx.y >= n_items) {
    const int at = blockIdx.y - n_items, i = at / blocks;
    decode_share<FMT, D>(p, blockIdx.x, prefix, counts, B, shares, i, at - i * blocks, static_cast<int64_t>(B) * p.Hq * slots, space,
                         reinterpret_cast<float(*)[16]>(m_lds), reinterpret_cast<float(*)[16]>(l_lds));
    return;
  }
  const int32_t* it = items + blockIdx.y * 8;
  RowsBlock w;
  w.tok0 = w.table = it[0];
  w.ntok = it[1];
  w.block = it[2];
  w.kend = min(it[4], p.width * p.bs);
  w.kbeg = min(it[3], w.kend);
  if (w.kbeg >= w.kend) w.kbeg = w.kend = 0;
  w.whole = false;
  w.part0 = it[5];
  w.part_step = slots;
  w.causal0 = OWN;
  if constexpr (RT == 8) attend_block<FMT, D>(p, w, blockIdx.x, space);
  else attend_rows<FMT, D, RT, false>(p, w, blockIdx.x, space, m_lds, l_lds);
}

// Joins a row's parts: out = sum_s 2^(lse_s - M) part_s / sum_s 2^(lse_s - M). They are the first counts[token] (null: all) of the
// row's `slots`, and, of `shares`, its sequence's; rows of one part are in `out` already. qsl: tokens outside [qsl[0], qsl[S]) have
// none. A workgroup has ROWS rows of a token, four dims a thread, and 4 x 1024 / (D ROWS) parts of a row on their way at once: one row
// where there are few (72 rows of 57 parts took 8.3 us with D / 4 threads a row), four where workgroups would only queue. Factors are
// 2^-8 of these at most: up to 256 parts' sums of the largest numbers stay numbers.
struct JoinArgs {
  const int32_t* counts;
  int slots;
  const int32_t* starts;
  int B, shares;
  const int32_t* qsl;
  int S;
};
template <int D, int ROWS>
__global__ void __launch_bounds__(256) rows_join_kernel(RowsArgs p, JoinArgs j) {
  constexpr int TPR = D / 4, GROUPS = 256 / TPR, OF_ROW = GROUPS / ROWS, AHEAD = 4;
  __shared__ float sums[GROUPS], tops[GROUPS];
  __shared__ __attribute__((aligned(16))) float outs[GROUPS][D];
  const int tok = blockIdx.x;
  if (j.qsl && (tok < j.qsl[0] || tok >= j.qsl[j.S])) return;
  const int d = threadIdx.x % TPR * 4, group = threadIdx.x / TPR, mine = group % OF_ROW;
  const int head = blockIdx.y * ROWS + group / OF_ROW;
  const int front = j.counts ? min(max(j.counts[tok], 0), j.slots) : j.slots;
  int n = front, first = 0;
  if (j.shares) {
    const Share s = find_share(p, j.starts, j.B, j.shares, 0, tok);
    n += s.parts;
    first = s.first;
    if (n == 1) return;
  }
  const int64_t row = static_cast<int64_t>(tok) * p.Hq + min(head, p.Hq - 1);
  const int64_t back = (static_cast<int64_t>(j.B) * j.slots + first) * p.Hq + min(head, p.Hq - 1);
  float M = LOWEST, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = mine; i0 < n; i0 += AHEAD * OF_ROW) {
    float e[AHEAD], top = M;
    float4 x[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = min(i0 + a * OF_ROW, n - 1);
      const int64_t part = i < front ? row * j.slots + i : back + static_cast<int64_t>(i - front) * p.Hq;
      e[a] = p.part_lse[part];
      x[a] = *reinterpret_cast<const float4*>(p.part_out + part * D + d);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i0 + a * OF_ROW >= n) {   // (read once more: 0 times an infinity of it would be NaN)
        e[a] = -INFINITY;
        x[a] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      top = fmaxf(top, e[a]);
    }
    const float old = exp2_fast(M - top);
    M = top;
    sum *= old;
    o = make_float4(o.x * old, o.y * old, o.z * old, o.w * old);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const float f = exp2_fast(e[a] - M - 8.f);
      sum += f;
      o = make_float4(o.x + f * x[a].x, o.y + f * x[a].y, o.z + f * x[a].z, o.w + f * x[a].w);
    }
  }
  if (d == 0) {
    sums[group] = sum;
    tops[group] = M;
  }
  *reinterpret_cast<float4*>(&outs[group][d]) = o;
  __syncthreads();
  if (mine != 0 || head >= p.Hq) return;
#pragma unroll
  for (int i = 1; i < OF_ROW; ++i) M = fmaxf(M, tops[group + i]);
  sum = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < OF_ROW; ++i) {
    const float f = exp2_fast(tops[group + i] - M);
    const float4 x = *reinterpret_cast<const float4*>(&outs[group + i][d]);
    sum += sums[group + i] * f;
    o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(p.out + tok * p.out_stride + static_cast<int64_t>(head) * D + d) =
      make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
}

static bool rows_ok(const RowsArgs& p, int D) {
  return p.bs > 0 && p.bs % KV_TILE == 0 && p.Hkv >= 1 && p.Hq % p.Hkv == 0 && (D == 64 || D == 128) && p.width >= 1 &&
         p.num_blocks >= 1 && !p.part_out == !p.part_lse && p.q_stride % 8 == 0 &&
         p.out_stride % 4 == 0 && static_cast<int64_t>(p.width) * (p.bs / KV_TILE) * (p.bs / KV_TILE) < 1 << 30 &&
         static_cast<int64_t>(p.width) * p.bs < 1ll << 31 && static_cast<int64_t>(p.Hkv) * p.bs * D < 1ll << 31;
}
static uint32_t page_magic(int bs) { return bs >= KV_TILE ? (1u << 31) / (bs / KV_TILE) + 1 : 1; }

static void join(const RowsArgs& p, int D, int tokens, const JoinArgs& j, hipStream_t st) {
  const bool few = static_cast<int64_t>(tokens) * p.Hq <= 512;
  const dim3 grid(tokens, few ? p.Hq : (p.Hq + 3) / 4);
  if (D == 128 && few) hipLaunchKernelGGL((rows_join_kernel<128, 1>), grid, dim3(256), 0, st, p, j);
  else if (D == 128) hipLaunchKernelGGL((rows_join_kernel<128, 4>), grid, dim3(256), 0, st, p, j);
  else if (few) hipLaunchKernelGGL((rows_join_kernel<64, 1>), grid, dim3(256), 0, st, p, j);
  else hipLaunchKernelGGL((rows_join_kernel<64, 4>), grid, dim3(256), 0, st, p, j);
}

#define XGK_FMT_DIM(DO)                                                                                              \
  if (fmt == KV_FP8 && D == 128) DO(KV_FP8, 128) else if (fmt == KV_FP8) DO(KV_FP8, 64)                               \
  else if (fmt == KV_INT8 && D == 128) DO(KV_INT8, 128) else if (fmt == KV_INT8) DO(KV_INT8, 64)

// Decode over an 8-bit cache. shares: B (whole rows), or more (part_out / part_lse: shares Hq parts). Returns 0, or -1 for what it
// does not take.
int quant_decode_attention(int fmt, const uint16_t* q, int64_t q_stride, const uint8_t* k, const uint8_t* v, const float* scales,
                           const int32_t* tables, int64_t table_stride, int width, const int32_t* seq_lens, float* part_out,
                           float* part_lse, uint16_t* out, int64_t out_stride, int B, int Hq, int Hkv, int D, int bs,
                           int num_blocks, float scale, int shares, int least, hipStream_t st) {
  if (B <= 0) return 0;
  const RowsArgs p{q, q_stride, k, v, scales, tables, table_stride, width, num_blocks, seq_lens, part_out, part_lse, out,
                   out_stride, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, bs, scale * 1.44269504088896341f, page_magic(bs), least};
  const int blocks = (p.G + 15) / 16;
  if (!rows_ok(p, D) || least < 1 || shares < B || static_cast<int64_t>(shares) * blocks > 65535 || (shares > B) != (part_out != nullptr)) return -1;
#define XGK_GO(F, DD)                                                                                                        \
  {                                                                                                                          \
    hipLaunchKernelGGL((rows_decode_kernel<F, DD>), dim3(Hkv, shares * blocks), dim3(256), 0, st, p, B, blocks, shares);     \
  }
  XGK_FMT_DIM(XGK_GO) else return -1;
#undef XGK_GO
  if (part_out) join(p, D, B, JoinArgs{nullptr, 0, nullptr, B, shares, nullptr, 0}, st);
  return 0;
}

// Causal attention of packed prompt portions over an 8-bit cache; 16 RT rows a workgroup, `splits` parts of their keys (parts:
// tokens Hq splits).
int quant_prefill_attention(int fmt, const uint16_t* q, int64_t q_stride, const uint8_t* k, const uint8_t* v, const float* scales,
                            const int32_t* tables, int64_t table_stride, int width, const int32_t* qsl, const int32_t* seq_lens,
                            float* part_out, float* part_lse, uint16_t* out, int64_t out_stride, int tokens, int S, int max_q,
                            int Hq, int Hkv, int D, int bs, int num_blocks, float scale, int RT, int splits, hipStream_t st) {
  if (tokens <= 0 || S <= 0 || max_q <= 0) return 0;
  const RowsArgs p{q, q_stride, k, v, scales, tables, table_stride, width, num_blocks, seq_lens, part_out, part_lse, out,
                   out_stride, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, bs, scale * 1.44269504088896341f, page_magic(bs), 1};
  if (!rows_ok(p, D) || (RT != 1 && RT != 2 && RT != 8) || splits < 1 || (splits > 1) != (part_out != nullptr)) return -1;
  const int64_t blocks = (static_cast<int64_t>(max_q) * p.G + 16 * RT - 1) / (16 * RT);
  if (blocks > 65535 || static_cast<int64_t>(S) * splits > 65535) return -1;
  const dim3 grid(Hkv, static_cast<unsigned>(blocks), S * splits);
#define XGK_GO(F, DD)                                                                                                        \
  {                                                                                                                          \
    if (RT == 1) hipLaunchKernelGGL((rows_prompt_kernel<F, DD, 1>), grid, dim3(256), 0, st, p, qsl, tokens, splits);         \
    else if (RT == 2) hipLaunchKernelGGL((rows_prompt_kernel<F, DD, 2>), grid, dim3(256), 0, st, p, qsl, tokens, splits);    \
    else hipLaunchKernelGGL((rows_prompt_kernel<F, DD, 8>), grid, dim3(256), 0, st, p, qsl, tokens, splits);                 \
  }
  XGK_FMT_DIM(XGK_GO) else return -1;
#undef XGK_GO
  if (part_out) join(p, D, tokens, JoinArgs{nullptr, splits, nullptr, 0, 0, qsl, S}, st);
  return 0;
}

// Decode rows in groups with a common prefix. items: rows_shared_kernel's, prefix: keys of each row that the items cover, counts: its
// parts of them (at most `slots`), shares: of the keys behind. Whole rows where slots is 0 and shares B; else B Hq slots + shares Hq
// parts.
int shared_prefix_attention(int fmt, const uint16_t* q, int64_t q_stride, const void* k, const void* v, const float* scales,
                            const int32_t* tables, int64_t table_stride, int width, const int32_t* seq_lens, float* part_out,
                            float* part_lse, uint16_t* out, int64_t out_stride, int B, int Hq, int Hkv, int D, int bs,
                            int num_blocks, float scale, const int32_t* items, int n_items, const int32_t* prefix,
                            const int32_t* counts, int slots, int RT, int shares, int least, hipStream_t st) {
  if (B <= 0) return 0;
  const RowsArgs p{q, q_stride, static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), scales, tables, table_stride,
                   width, num_blocks, seq_lens, part_out, part_lse, out, out_stride, Hq, Hkv, Hkv > 0 ? Hq / Hkv : 0, bs,
                   scale * 1.44269504088896341f, page_magic(bs), least};
  const int blocks = (p.G + 15) / 16;
  if (!rows_ok(p, D) || least < 1 || (RT != 1 && RT != 2 && RT != 8) || shares < B || slots < 0 || n_items < 0 ||
      n_items + static_cast<int64_t>(shares) * blocks > 65535 || (slots > 0 || shares > B) != (part_out != nullptr))
    return -1;
  const dim3 grid(Hkv, n_items + shares * blocks);
#define XGK_SHARED(F, DD, R)                                                                                                   \
  hipLaunchKernelGGL((rows_shared_kernel<F, DD, R>), grid, dim3(256), 0, st, p, items, n_items, prefix, counts, slots, B, blocks, shares)
#define XGK_GO(F, DD)                           \
  {                                             \
    if (RT == 1) XGK_SHARED(F, DD, 1);          \
    else if (RT == 2) XGK_SHARED(F, DD, 2);     \
    else return -1;                             \
  }
  XGK_FMT_DIM(XGK_GO)
  else if (fmt == KV_BF16 && RT == 8) {
    if (D == 128) XGK_SHARED(KV_BF16, 128, 8);
    else XGK_SHARED(KV_BF16, 64, 8);
  }
  else if (fmt == KV_BF16 && D == 128) XGK_GO(KV_BF16, 128) else if (fmt == KV_BF16) XGK_GO(KV_BF16, 64) else return -1;
#undef XGK_GO
#undef XGK_SHARED
  if (part_out) join(p, D, B, JoinArgs{counts, slots, prefix, B, shares, nullptr, 0}, st);
  return 0;
}

}  // namespace xgk
