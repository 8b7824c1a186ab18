// Writing the 8-bit paged KV cache (kv_quant.h) and reading it back.
#include "kv_quant.h"

namespace xgk {

// ---- append ------------------------------------------------------------------------------------------------------------
// A wave takes a window of four tokens of one head (or two): 16 lanes a row, D / 16 numbers a lane, K and V in turn. A row's largest
// magnitude joins over its 16 lanes by register rotations; nothing goes through memory but the row itself (2 D bytes in,
// D + 4 out: bound by HBM for long steps, by one trip to memory and the launch for single tokens).
//
// Codes as the mathematics has them: with bf16 x and a, the distance of 127 x / a (448 x / a) from the border of two codes
// is 0 or at least 2^-16 of it, so x (127 / a), off by less than 2^-22, rounded to 20 bits is on the border exactly when
// the quotient is, and rounds to even there.
//
// V's order puts four tokens' codes of a dim into one word: a window whose slots fill such a quad (tokens of a prompt)
// exchanges its codes within the wave and writes words; other tokens write bytes.
//
// Where the rows come from: KV_ROWS k and v as they are; KV_ROPE the rows of the QKV projection, q and k rotated; KV_PARTS the
// projection's split-K partial sums [S, T, (Hq + 2 Hkv) D] in fp32, added up, q and k rotated (with a table) and rounded to bf16.
enum : int { KV_ROWS = 0, KV_ROPE = 1, KV_PARTS = 2 };
struct KvAppend {
  uint16_t* q;                 // query heads: KV_ROPE in place (tokens as k's), KV_PARTS written to
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_stride, v_stride;  // elements between tokens
  const float* part;           // KV_PARTS
  int S;
  int64_t q_stride;
  const int32_t* slots;        // slot of each token; outside [0, num_slots): not written
  const int32_t* positions;    // of a rotation
  const float* cos_sin;        // [max_pos, D]
  uint8_t* kc;
  uint8_t* vc;
  float* scales;
  int64_t num_slots;
  int T, Hq, Hkv, bs;
};

template <int N>
struct Codes { uint32_t w[N / 4]; };

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// codes of this lane's D / 16 numbers (N / 2 pairs) of a row that 16 lanes hold, and the row's scale
template <int FMT, int N>
__device__ __forceinline__ Codes<N> kv_quantise(const uint32_t (&x)[N / 2], float& scale) {
  constexpr float LARGEST = FMT == KV_FP8 ? 448.f : 127.f;
  // magnitudes of bf16 order as whole numbers do, NaN above infinity
  u16x2_t pair = {0, 0};
#pragma unroll
  for (int i = 0; i < N / 2; ++i) pair = __builtin_elementwise_max(pair, __builtin_bit_cast(u16x2_t, x[i] & 0x7FFF7FFFu));
  uint32_t top = max(pair[0], pair[1]);
  auto join = [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); };
  float m = __uint_as_float(top);
  m = join(m, row_ror<8>(m));
  m = join(m, row_ror<4>(m));
  m = join(m, row_ror<2>(m));
  m = join(m, row_ror<1>(m));
  top = __float_as_uint(m);
  float a = __uint_as_float(top << 16);
  float y[N];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    y[2 * i] = __uint_as_float(x[i] << 16);
    y[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
  }
  if (__all(a > 0x1p-90f && a < 0x1p100f)) {
    // a / LARGEST to its nearest float: the quotient's own error comes back through the multiply-add
    const float q = a * (1.f / LARGEST);
    scale = fmaf(fmaf(-LARGEST, q, a), 1.f / LARGEST, q);
  } else {   // rows of zeros, of numbers whose inverse is no normal float, and those that are not finite
    const bool usable = top < 0x7F80u && top != 0;
    scale = usable ? a / LARGEST : (top == 0 ? 0.f : __uint_as_float(0x7FC00000u));
    const float lift = a >= 0x1p100f ? 0x1p-60f : a > 0x1p-90f ? 1.f : 0x1p60f;
    a = usable ? a * lift : 1.f;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = usable ? y[i] * lift : 0.f;
  }
#if defined(__HIP_DEVICE_COMPILE__)
  const float inv = LARGEST * __builtin_amdgcn_rcpf(a);   // off by less than 2^-22.4, the products by less than 2^-22
#else
  const float inv = LARGEST / a;
#endif
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = __uint_as_float((__float_as_uint(y[i] * inv) + 8u) & ~15u);
  Codes<N> c;
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (FMT == KV_FP8) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], w, true);
      c.w[j] = static_cast<uint32_t>(w);
    } else {
      // 1.5 2^23 more: the float's last byte is the whole number, rounded to even, in two's complement
      uint32_t e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = __float_as_uint(y[4 * j + i] + 12582912.f);
      c.w[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(e[3], e[2], 0x0C0C0400u), __builtin_amdgcn_perm(e[1], e[0], 0x0C0C0400u), 0x05040100u);
    }
#else
    c.w[j] = 0;
#endif
  }
  return c;
}

template <int N>
__device__ __forceinline__ void kv_load_row(const uint16_t* p, uint32_t (&x)[N / 2]) {
  if constexpr (N == 8) {
    const uint4 v = ld16(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = v.x; x[1] = v.y;
  }
}

// Codes of four tokens, a token a 16-lane group, to words of four tokens' codes of a dim: group i has the dims (N / 4) i + e of its N.
// Halves of the wave trade places, then neighbouring groups: two register moves where a trip through LDS a word was eight.
template <int N>
__device__ __forceinline__ void kv_turn(const Codes<N>& c, uint32_t (&four)[N / 4]) {
#if defined(__HIP_DEVICE_COMPILE__)
  // lo / hi: the N / 2 codes of the lower and upper dims. Behind the first move the lower groups have tokens' (0 | 1) and (2 | 3) lo
  const uint32_t lo = N == 8 ? c.w[0] : c.w[0] & 0xFFFFu, hi = N == 8 ? c.w[N / 4 - 1] : c.w[0] >> 16;
  const auto h = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
  // of these the first and second halves, tokens (0 | 1) below (2 | 3)
  const uint32_t x = __builtin_amdgcn_perm(h[1], h[0], N == 8 ? 0x05040100u : 0x0C0C0400u);
  const uint32_t y = __builtin_amdgcn_perm(h[1], h[0], N == 8 ? 0x07060302u : 0x0C0C0501u);
  const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);   // tokens 0, 2 and 1, 3 of the group's own dims
  if constexpr (N == 8) {
    four[0] = __builtin_amdgcn_perm(r[1], r[0], 0x06020400u);
    four[N / 4 - 1] = __builtin_amdgcn_perm(r[1], r[0], 0x07030501u);
  } else {
    four[0] = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u);
  }
#endif
}

// rotate_half of a row that 16 lanes hold: lane c's partner is c ^ 8 (D / 2 numbers on)
template <int N>
__device__ __forceinline__ void kv_rotate(float (&f)[N], const float* cs, int c) {
  const float* cp = cs + (c & 7) * N;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float o = row_ror<8>(f[i]), co = cp[i], si = cp[8 * N + i];
    f[i] = c < 8 ? f[i] * co - o * si : f[i] * co + o * si;
  }
}

// N numbers of a token's partial sums, added up: four parts' loads at a time
template <int N>
__device__ __forceinline__ void kv_sum_parts(const float* p, int S, int64_t slab, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = 0.f;
  for (int s0 = 0; s0 < S; s0 += 4) {
    float4 x[4][N / 4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < N / 4; ++i) x[j][i] = *reinterpret_cast<const float4*>(p + min(s0 + j, S - 1) * slab + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float on = s0 + j < S ? 1.f : 0.f;
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        f[4 * i] += on * x[j][i].x; f[4 * i + 1] += on * x[j][i].y; f[4 * i + 2] += on * x[j][i].z; f[4 * i + 3] += on * x[j][i].w;
      }
    }
  }
}

template <int FMT, int D, int FROM, int HEADS>
__global__ void __launch_bounds__(256) kv_append_kernel(KvAppend p) {
  constexpr int N = D / 16;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = (blockIdx.x * 4 + wid) * 4, head = blockIdx.y * HEADS;
  const int i = lane >> 4, c = lane & 15;
  if (t0 >= p.T) return;
  // this lane's numbers of a row, as bf16 pairs: `at` the row's, `column` its place in the partial sums
  auto row = [&](const uint16_t* at, int64_t column, int t, bool turn, uint32_t (&x)[N / 2]) {
    if constexpr (FROM != KV_PARTS) kv_load_row<N>(at + c * N, x);
    if constexpr (FROM != KV_ROWS) {
      float f[N];
      if constexpr (FROM == KV_PARTS) {
        const int64_t width = static_cast<int64_t>(p.Hq + 2 * p.Hkv) * D;
        kv_sum_parts<N>(p.part + t * width + column + c * N, p.S, p.T * width, f);
      } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          f[2 * j] = __uint_as_float(x[j] << 16);
          f[2 * j + 1] = __uint_as_float(x[j] & 0xFFFF0000u);
        }
      }
      if (turn && p.cos_sin) kv_rotate<N>(f, p.cos_sin + static_cast<int64_t>(p.positions[t]) * D, c);
#pragma unroll
      for (int j = 0; j < N / 2; ++j) x[j] = pack2(f[2 * j], f[2 * j + 1]);
    }
  };
  if (FROM != KV_ROWS && head >= p.Hkv) {   // a query head
    const int t = t0 + i, h = head - p.Hkv;
    if (t < p.T) {
      uint16_t* dst = p.q + static_cast<int64_t>(t) * p.q_stride + static_cast<int64_t>(h) * D;
      uint32_t x[N / 2];
      row(dst, static_cast<int64_t>(h) * D, t, true, x);
      if constexpr (N == 8) st16(dst + c * N, make_uint4(x[0], x[1], x[N / 2 - 2], x[N / 2 - 1]));
      else *reinterpret_cast<uint2*>(dst + c * N) = make_uint2(x[0], x[1]);
    }
    return;
  }
  // slots of the tokens around the window, -1 where there is none
  int s[10];
#pragma unroll
  for (int j = 0; j < 10; ++j) {
    const int t = t0 - 3 + j;
    const int v = p.slots[min(max(t, 0), p.T - 1)];
    s[j] = t >= 0 && t < p.T && static_cast<int64_t>(v) < p.num_slots ? v : -1;
  }
  // the quad that begins in this window, and this window's tokens that no quad takes
  int quad = -1, quad_slot = 0;
  uint32_t taken = 0;
#pragma unroll
  for (int b = 0; b < 7; ++b)
    if (s[b] >= 0 && (s[b] & 3) == 0 && s[b + 1] == s[b] + 1 && s[b + 2] == s[b] + 2 && s[b + 3] == s[b] + 3) {
      if (b >= 3) {
        quad = t0 - 3 + b;
        quad_slot = s[b];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b + j >= 3 && b + j < 7) taken |= 1u << (b + j - 3);
    }
  // the 16 lanes' token t at offset `off` of a page: its codes of K and V
  auto write = [&](int t, int64_t page, int off, bool whole) {
    uint32_t xk[HEADS][N / 2], xv[HEADS][N / 2];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int64_t dim = static_cast<int64_t>(head + h) * D;
      row(p.k + static_cast<int64_t>(t) * p.k_stride + dim, static_cast<int64_t>(p.Hq) * D + dim, t, true, xk[h]);
      row(p.v + static_cast<int64_t>(t) * p.v_stride + dim, static_cast<int64_t>(p.Hq + p.Hkv) * D + dim, t, false, xv[h]);
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int64_t ph = page * p.Hkv + head + h, tile = (ph * p.bs + (off & ~15)) * D, at = ph * 2 * p.bs + off;
      float sk, sv;
      const Codes<N> wk = kv_quantise<FMT, N>(xk[h], sk), wv = kv_quantise<FMT, N>(xv[h], sv);
      uint8_t* dk = p.kc + tile + kv_k_byte(off & 15, c * N);
      if constexpr (N == 8) *reinterpret_cast<uint2*>(dk) = make_uint2(wk.w[0], wk.w[N / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(dk) = wk.w[0];
      if (c == 0) {
        p.scales[at] = sk;
        p.scales[at + p.bs] = sv;
      }
      if (whole) {
        uint32_t four[N / 4];
        kv_turn<N>(wv, four);
#pragma unroll
        for (int e = 0; e < N / 4; ++e)
          *reinterpret_cast<uint32_t*>(p.vc + tile + kv_v_byte(off & 12, c * N + (N / 4) * i + e)) = four[e];
      } else {
        uint8_t* dv = p.vc + tile + kv_v_byte(off & 15, c * N);
#pragma unroll
        for (int e = 0; e < N; ++e) dv[16 * e] = (wv.w[e >> 2] >> (8 * (e & 3))) & 0xFF;
      }
    }
  };
  if (quad >= 0) {   // (one division for the wave)
    const int page = quad_slot / p.bs;
    write(quad + i, page, quad_slot - page * p.bs + i, true);
  }
  const int slot = i == 0 ? s[3] : i == 1 ? s[4] : i == 2 ? s[5] : s[6];
  if (!(taken >> i & 1) && slot >= 0)   // (16 lanes are of one mind: the rotations within them stay whole)
    write(t0 + i, slot / p.bs, slot % p.bs, false);
}

template <int FMT, int D>
static void launch_append(const KvAppend& p, int from, hipStream_t st) {
  const dim3 grid((p.T + 15) / 16, p.Hkv + (from != KV_ROWS ? p.Hq : 0));
  // two heads a wave from 16 k rows on: half the waves, each with twice the loads on their way, 14.5 -> 11.5 us for 8192 tokens of 8
  // heads and 46 -> 34 (6 TB/s) for 32768, the same rows each time (in turn with others 11.8 and 42); 4.0 for 3.5 with 64 tokens, where
  // they are too few
  if (from == KV_PARTS) hipLaunchKernelGGL((kv_append_kernel<FMT, D, KV_PARTS, 1>), grid, dim3(256), 0, st, p);
  else if (from == KV_ROPE) hipLaunchKernelGGL((kv_append_kernel<FMT, D, KV_ROPE, 1>), grid, dim3(256), 0, st, p);
  else if (p.Hkv % 2 == 0 && static_cast<int64_t>(p.T) * p.Hkv >= 16384)
    hipLaunchKernelGGL((kv_append_kernel<FMT, D, KV_ROWS, 2>), dim3(grid.x, p.Hkv / 2), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((kv_append_kernel<FMT, D, KV_ROWS, 1>), grid, dim3(256), 0, st, p);
}

static int append(int fmt, const KvAppend& p, int from, int D, hipStream_t st) {
  if (p.T <= 0) return 0;
  if (p.bs <= 0 || p.bs % KV_TILE || p.Hkv < 1 || (D != 64 && D != 128)) return -1;
  if (fmt == KV_FP8 && D == 128) launch_append<KV_FP8, 128>(p, from, st);
  else if (fmt == KV_FP8) launch_append<KV_FP8, 64>(p, from, st);
  else if (fmt == KV_INT8 && D == 128) launch_append<KV_INT8, 128>(p, from, st);
  else if (fmt == KV_INT8) launch_append<KV_INT8, 64>(p, from, st);
  else return -1;
  return 0;
}

// cos_sin null: k and v as they are; else q (Hq heads, in place) and k are rotated first.
int kv_append(int fmt, uint16_t* q, const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride,
              const int32_t* slots, const int32_t* positions, const float* cos_sin, uint8_t* kc, uint8_t* vc, float* scales,
              int64_t num_blocks, int T, int Hq, int Hkv, int D, int bs, hipStream_t st) {
  if (k_stride % (D >= 16 ? D / 16 : 1) || v_stride % (D >= 16 ? D / 16 : 1)) return -1;
  if (cos_sin != nullptr && (q == nullptr || positions == nullptr)) return -1;
  const KvAppend p{q, k, v, k_stride, v_stride, nullptr, 0, k_stride, slots, positions, cos_sin, kc, vc, scales, num_blocks * bs,
                   T, Hq, Hkv, bs};
  return append(fmt, p, cos_sin ? KV_ROPE : KV_ROWS, D, st);
}

// The same of partial sums; q goes to q_out. cos_sin null: no rotation.
int kv_append_partials(int fmt, const float* part, int S, uint16_t* q_out, int64_t q_stride, const int32_t* slots,
                       const int32_t* positions, const float* cos_sin, uint8_t* kc, uint8_t* vc, float* scales,
                       int64_t num_blocks, int T, int Hq, int Hkv, int D, int bs, hipStream_t st) {
  if (S < 1 || part == nullptr || q_out == nullptr || q_stride % 8 || (cos_sin != nullptr && positions == nullptr)) return -1;
  const KvAppend p{q_out, nullptr, nullptr, 0, 0, part, S, q_stride, slots, positions, cos_sin, kc, vc, scales, num_blocks * bs,
                   T, Hq, Hkv, bs};
  return append(fmt, p, KV_PARTS, D, st);
}

// ---- read back ---------------------------------------------------------------------------------------------------------
// Tokens starts[s] + i, i < cu[s + 1] - cu[s], of every sequence as bf16 rows [n, Hkv, D]. A wave takes one 16-token tile of
// one head: two (D = 128) whole 1 KiB reads of K and of V, widened, scaled and put in rows through LDS (V's codes come in
// token quads a dim), written as 16 bytes a lane. (D + 4) bytes in and 2 D out a row: bound by HBM.
// Tile j of the launch belongs to the last sequence s with cu[s] / 16 + 2 s <= j: n tokens that begin anywhere in a tile
// touch at most n / 16 + 2 of them.
template <int FMT, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                      const float* __restrict__ scales,
                                                      const int32_t* __restrict__ tables, int64_t table_stride, int width,
                                                      const int32_t* __restrict__ starts, const int32_t* __restrict__ cu,
                                                      int S, int n, int num_blocks, int Hkv, int bs, uint16_t* __restrict__ k,
                                                      uint16_t* __restrict__ v) {
  constexpr int ROW = D + 8;      // LDS row, padded: 16 rows of a column fall on different banks
  constexpr int LOADS = D / 64;
  __shared__ __attribute__((aligned(16))) uint16_t rows[4][16 * ROW];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, li = lane & 15;
  const int j = blockIdx.x * 4 + wid, head = blockIdx.y;
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] / 16 + 2 * mid <= j) lo = mid;
    else hi = mid - 1;
  }
  const int first = starts[lo], out0 = cu[lo], count = min(cu[lo + 1], n) - out0;
  const int ahead = j - (out0 / 16 + 2 * lo);
  if (count <= 0 || first < 0 || out0 < 0 || ahead < 0) return;
  const int tile = (first >> 4) + ahead;
  // (tiles behind the sequence's end, or behind its table's: nothing to do)
  if (tile * 16 >= first + count || tile >= width * (bs >> 4)) return;
  const int page = min(max(tables[lo * table_stride + tile * 16 / bs], 0), num_blocks - 1);
  const int off = tile * 16 % bs;
  const int64_t ph = static_cast<int64_t>(page) * Hkv + head;
  const int64_t base = (ph * bs + off) * D;
  const float* sc = scales + ph * 2 * bs + off;
  uint4 kr[LOADS], vr[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    kr[i] = ld16_nt(kc + base + i * 1024 + lane * 16);
    vr[i] = ld16_nt(vc + base + i * 1024 + lane * 16);
  }
  const float ks = sc[li];
  const float4 vs4 = *reinterpret_cast<const float4*>(sc + bs + 4 * g);
  const float vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};
  uint16_t* mine = rows[wid];
  auto emit = [&](uint16_t* dst) {   // (a wave's own rows: its LDS writes and reads are in order)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int ch = lane + 64 * i, t = ch / (D / 8), at = tile * 16 + t - first;
      const uint4 w = ld16(mine + t * ROW + ch % (D / 8) * 8);
      if (at >= 0 && at < count) st16(dst + ((static_cast<int64_t>(out0) + at) * Hkv + head) * D + ch % (D / 8) * 8, w);
    }
    __builtin_amdgcn_wave_barrier();
  };
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const uint32_t w[4] = {kr[i].x, kr[i].y, kr[i].z, kr[i].w};
    uint32_t o[8];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint2 b = kv_widen4<FMT>(w[x]);
      o[2 * x] = pack2(__uint_as_float(b.x << 16) * ks, __uint_as_float(b.x & 0xFFFF0000u) * ks);
      o[2 * x + 1] = pack2(__uint_as_float(b.y << 16) * ks, __uint_as_float(b.y & 0xFFFF0000u) * ks);
    }
    uint16_t* dst = mine + li * ROW + 16 * (4 * i + g);
    st16(dst, make_uint4(o[0], o[1], o[2], o[3]));
    st16(dst + 8, make_uint4(o[4], o[5], o[6], o[7]));
  }
  emit(k);
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint2 b = kv_widen4<FMT>(w[x]);
      const int d = 64 * i + 16 * x + li;
      mine[(4 * g + 0) * ROW + d] = f2bf(__uint_as_float(b.x << 16) * vs[0]);
      mine[(4 * g + 1) * ROW + d] = f2bf(__uint_as_float(b.x & 0xFFFF0000u) * vs[1]);
      mine[(4 * g + 2) * ROW + d] = f2bf(__uint_as_float(b.y << 16) * vs[2]);
      mine[(4 * g + 3) * ROW + d] = f2bf(__uint_as_float(b.y & 0xFFFF0000u) * vs[3]);
    }
  }
  emit(v);
}

int kv_read(int fmt, const uint8_t* kc, const uint8_t* vc, const float* scales, const int32_t* tables, int64_t table_stride,
            int width, const int32_t* starts, const int32_t* cu, int S, int n, int num_blocks, int Hkv, int D, int bs,
            uint16_t* k, uint16_t* v, hipStream_t st) {
  if (S <= 0 || n <= 0) return 0;
  if (bs <= 0 || bs % KV_TILE || Hkv < 1 || num_blocks < 1 || width < 1) return -1;
  const dim3 grid((n / 16 + 2 * S + 3) / 4, Hkv);
#define XGK_READ(F, DD)                                                                                                  \
  if (fmt == F && D == DD) {                                                                                             \
    hipLaunchKernelGGL((kv_read_kernel<F, DD>), grid, dim3(256), 0, st, kc, vc, scales, tables, table_stride, width,     \
                       starts, cu, S, n, num_blocks, Hkv, bs, k, v);                                                     \
    return 0;                                                                                                            \
  }
  XGK_READ(KV_FP8, 128) XGK_READ(KV_FP8, 64) XGK_READ(KV_INT8, 128) XGK_READ(KV_INT8, 64)
#undef XGK_READ
  return -1;
}

}  // namespace xgk
