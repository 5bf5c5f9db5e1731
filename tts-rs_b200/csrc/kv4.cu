// Operators of the 4-bit paged key/value cache: append (q/k RMSNorm, rotary
// positions, quantisation), attend (causal GQA over the cache) and read.
//
// A group of 32 values x is stored as digits n in 0..15 with bf16 scale s and
// zero z:  z = min(x) rounded down, s = bf16((max(x) - z) / 15),
// n = round((x - z) / s);  it stands for n s + z, within s / 2 of x.
//
// Block of one (page of 16 tokens, kv head), D = head_dim, G = D / 32 groups
// (every byte belongs to one token, so tokens append without reading):
//   K digits  [token c][t 4][group j][4 bytes]: dim 32 j + 8 t + 4 b0 + 2 h +
//             b1 in nibble h of byte 2 b1 + b0
//   V digits  [D / 64][g 8][t 4][m 4][4 bytes]: token 8 b0 + 2 t + b1, dim
//             64 M + 16 m + 8 h + g in nibble h of byte 2 b1 + b0
//   scales    [group j][t 4][4]{Ks, Kz, Vs, Vz}: entry 2 p1 + p0 is token
//             8 p1 + 2 t + p0
// The orders are those of the m16n8k16 fragments: with w one 32-bit word of
// digits, w & 0x000f000f, w & 0x00f000f0 and the same of w >> 8 are four
// fragment registers.  Read as f16 they are the subnormals n 2^-24 and
// 16 n 2^-24, exact, so digits reach the tensor cores with one mask each and
// no arithmetic; the powers of two are undone once per row.
#include <cuda_fp16.h>

#include <atomic>
#include <cfloat>
#include <cmath>

#include "common.cuh"
#include "engine.h"
#include "kv4.cuh"
#include "umma.cuh"

namespace q3t {

namespace {

// ---------------------------------------------------------------------------
// Which rows a CTA works on
// ---------------------------------------------------------------------------
// Token rows [t0, t0 + n) of sequence s, clamped to the call's rows; the
// last sits at position kv_len - 1.  (A length below 0 is as one of 0: all its
// rows are in front of position 0, and no position passes 32 bits.)
Q3T_DEV void seq_rows(const Kv4Batch &b, int s, int &t0, int &n, int &pos0) {
  const int lo = min(max(b.q_start[s], 0), b.num_tokens), hi = min(max(b.q_start[s + 1], lo), b.num_tokens);
  t0 = lo;
  n = hi - lo;
  pos0 = max(b.kv_len[s], 0) - n;
}

// Page of positions [16 p, 16 p + 16) of sequence s; -1 where the table or
// the pool has none.
Q3T_DEV int page_of(const Kv4View &c, const Kv4Batch &b, int s, int p) {
  const int row = b.table_row ? b.table_row[s] : b.first + s;
  if (p < 0 || p >= c.table_stride || row < 0 || row >= c.table_rows) return -1;
  const int id = c.table[(size_t)row * c.table_stride + p];
  return id >= 0 && id < c.num_pages ? id : -1;
}

// Items are numbered sequence by sequence, count(s) of them each; finds the
// sequence of `item` and its index there.  Block-wide; false past the end.
template <class F>
Q3T_DEV bool find_item(int num_seqs, int item, F count, int &s, int &i) {
  __shared__ int warp_tot[32], hit[2];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (num_seqs <= 128) {  // every warp for itself, four sequences to a lane
    int mine[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) mine[j] = 4 * lane + j < num_seqs ? count(4 * lane + j) : 0;
#pragma unroll
    for (int j = 0; j < 4; j++) sum += mine[j];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t found = __ballot_sync(0xffffffffu, item < incl);
    const int at = max(__ffs(found) - 1, 0);
    int j = 0, left = item - (incl - sum);  // of that lane's four: which, and where in it
#pragma unroll
    for (int x = 0; x < 3; x++)
      if (j == x && left >= mine[x]) left -= mine[x], j = x + 1;
    s = found ? 4 * at + __shfl_sync(0xffffffffu, j, at) : -1;
    i = __shfl_sync(0xffffffffu, left, at);
    return found != 0;
  }
  if (threadIdx.x == 0) hit[0] = -1;
  for (int base = 0; base < num_seqs; base += blockDim.x) {
    const int mine = base + (int)threadIdx.x < num_seqs ? count(base + threadIdx.x) : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) warp_tot[w] = incl;
    __syncthreads();
    int before = 0, total = 0;
    for (int k = 0; k < nw; k++) {
      if (k < w) before += warp_tot[k];
      total += warp_tot[k];
    }
    const int excl = before + incl - mine;
    if (item >= excl && item < excl + mine) {
      hit[0] = base + threadIdx.x;
      hit[1] = item - excl;
    }
    __syncthreads();
    if (hit[0] >= 0) break;
    item -= total;
  }
  s = hit[0];
  i = hit[1];
  return s >= 0;
}

// A window is the part of a sequence's rows that lies in one page: rows
// [t0, t0 + n) at slots c0 .. c0 + n - 1 of page index p.
struct Window {
  int s, t0, n, p, c0;
};
Q3T_DEV bool find_window(const Kv4Batch &b, int item, Window &w) {
  int i;
  const bool ok = find_item(
      b.num_seqs, item,
      [&](int s) {
        int t0, n, pos0;
        seq_rows(b, s, t0, n, pos0);
        return n > 0 ? ((pos0 + n - 1) >> 4) - (pos0 >> 4) + 1 : 0;
      },
      w.s, i);
  if (!ok) return false;
  int t0, n, pos0;
  seq_rows(b, w.s, t0, n, pos0);
  w.p = (pos0 >> 4) + i;  // negative for padding in front of position 0
  const int base = w.p * 16;
  w.c0 = max(pos0 - base, 0);
  w.t0 = t0 + base + w.c0 - pos0;
  w.n = min(pos0 + n - base, 16) - w.c0;
  return true;
}
// windows of a call, at most: a sequence's n rows touch (n + 14) / 16 + 1 pages, and n
int max_windows(const Kv4Batch &b) {
  const int64_t w = (int64_t)b.num_tokens / 16 + 2ll * b.num_seqs;
  return (int)(w < b.num_tokens ? w : b.num_tokens);
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
// Pairs of f32: one instruction for two of the same.
Q3T_DEV uint64_t f2_pack(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
Q3T_DEV void f2_split(uint64_t d, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
Q3T_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
Q3T_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
Q3T_DEV uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
Q3T_DEV uint64_t f2_sub(uint64_t a, uint64_t b) { return f2_fma(b, 0xbf800000bf800000ull, a); }

// Eight elements of a row, as they are and as floats.
template <typename T>
struct Raw8 {
  uint32_t w[2 * sizeof(T)];
};
template <typename T>
Q3T_DEV void load8(const T *p, bool vec, Raw8<T> &x) {
#pragma unroll
  for (int i = 0; i < (int)(2 * sizeof(T)); i += 4) {
    if (vec) {
      const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
      x.w[i] = u.x, x.w[i + 1] = u.y, x.w[i + 2] = u.z, x.w[i + 3] = u.w;
    } else {
#pragma unroll
      for (int k = i; k < i + 4; k++) {
        if constexpr (sizeof(T) == 4)
          x.w[k] = __float_as_uint(p[k]);
        else
          x.w[k] = p[2 * k] | (uint32_t)p[2 * k + 1] << 16;
      }
    }
  }
}
Q3T_DEV void floats(const Raw8<float> &x, float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = __uint_as_float(x.w[i]);
}
Q3T_DEV void floats(const Raw8<uint16_t> &x, float v[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[2 * i] = bf2f(x.w[i] & 0xffffu), v[2 * i + 1] = __uint_as_float(x.w[i] & 0xffff0000u);
}
Q3T_DEV void store8(uint16_t *p, bool vec, const float v[8]) {
  if (vec) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                               pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = f2bf(v[i]);
  }
}
// the smaller and the larger, NaN if one is
Q3T_DEV float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
Q3T_DEV float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Sum of squares to about 2^-45 of itself: every addition's error (Knuth's
// two-sum), and every square's, goes into a second sum.  In 32 bits, two at a
// time: a conversion to 64 costs as much as eight of these.  For sums in
// 2^-90 .. 2^100; another has squares that 32 bits do not hold.
template <int E>
Q3T_DEV double square_sum(const float (&v)[E][8]) {
  uint64_t sum = 0, rest = 0;
#pragma unroll
  for (int i = 0; i < 8 * E; i += 2) {
    const uint64_t x = f2_pack(v[i >> 3][i & 7], v[i >> 3][(i & 7) + 1]), sq = f2_mul(x, x);
    rest = f2_sub(rest, f2_fma(x, f2_mul(x, 0xbf800000bf800000ull), sq));
    if (i == 0) {
      sum = sq;
      continue;
    }
    const uint64_t t = f2_add(sum, sq), b = f2_sub(t, sum);
    rest = f2_add(rest, f2_add(f2_sub(sum, f2_sub(t, b)), f2_sub(sq, b)));
    sum = t;
  }
  float s0, s1, r0, r1;
  f2_split(sum, s0, s1);
  f2_split(rest, r0, r1);
  return (double)s0 + (double)s1 + (double)(r0 + r1);
}
// 1 / sqrt(x) rounded to 32 bits: the 32-bit one and a Newton step in 64 bits
Q3T_DEV float rsqrt64(double x) {
  const float f = (float)x;
  if (!(f > 0x1p-100f && f < 0x1p100f)) return (float)(1.0 / sqrt(x));
  const double y = rsqrtf(f), e = fma(-x * y, y, 1.0);
  return (float)fma(0.5 * e, y, y);
}

// Digits, scale and zero of a group of 32 that four lanes hold; a digit lies
// in the low bits of n[i], whose others are kDigit's.  A group with a value
// that is not finite gets a NaN scale and zero: it reads back as NaN, as such
// a value does from a cache that is not quantised.  Without a scale (false)
// the digits are to be zeros.
constexpr uint32_t kDigit = 0x4b400000u;  // 1.5 2^23
Q3T_DEV bool quantise(const float v[8], uint32_t n[8], uint32_t &scale_zero) {
  float lo = v[0], hi = v[0];
#pragma unroll
  for (int i = 1; i < 8; i++) lo = min_nan(lo, v[i]), hi = max_nan(hi, v[i]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const bool bad = !(fabsf(lo) <= FLT_MAX && fabsf(hi) <= FLT_MAX);
  // towards minus infinity: more magnitude below zero, less above
  uint32_t zb = __float_as_uint(lo);
  zb = ((zb >> 31 && (zb << 1)) ? zb + 0xffffu : zb) & 0xffff0000u;
  if (zb == 0xff800000u) zb = 0xff7f0000u;
  const float z = __uint_as_float(zb);
  // halves first: the range of two finite values need not be finite
  const uint16_t sb = f2bf(__fmul_rn(__fsub_rn(__fmul_rn(hi, 0.5f), __fmul_rn(z, 0.5f)), (float)(2.0 / 15.0)));
  const float s = bf2f(sb);
  scale_zero = bad ? 0x7fc07fc0u : sb | zb;
  // The quotient correctly rounded (Markstein 1990): y is 1 / s rounded, q the
  // product rounded, q + y (t - q s) then rounds as t / s does.  A scale that
  // is small enough for its reciprocal to overflow is first raised, with t.
  const float up = s < 0x1p-80f ? 0x1p100f : 1.f, su = s * up, y = __frcp_rn(su);
  const uint64_t z2 = f2_pack(-z, -z), up2 = f2_pack(up, up), s2 = f2_pack(-su, -su), y2 = f2_pack(y, y);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t t = f2_mul(f2_add(f2_pack(v[i], v[i + 1]), z2), up2), q = f2_mul(t, y2);
    float d0, d1;
    f2_split(f2_fma(f2_fma(q, s2, t), y2, q), d0, d1);
    d0 = fmaxf(fminf(d0, 15.f), 0.f), d1 = fmaxf(fminf(d1, 15.f), 0.f);  // (t infinite: 15)
    f2_split(f2_add(f2_pack(d0, d1), f2_pack(0x1.8p23f, 0x1.8p23f)), d0, d1);  // to the nearest, ties to even
    n[i] = __float_as_uint(d0), n[i + 1] = __float_as_uint(d1);
  }
  return !bad && s > 0.f;
}

// ---------------------------------------------------------------------------
// Append: one CTA per (window, head split).  A lane has eight dims of a row,
// four lanes a group of 32, and a warp two rows (D = 128) or four of one kind.
// Blocks are put together in shared memory, and a window that fills its page
// is written in 16-byte pieces, any other in the bytes that its tokens own.
// Bound by latency at few warps, not by bytes: a lane's 32 dims take 118
// registers, which leaves 16 warps to an SM, and these wait for fixed latencies,
// shuffles and shared memory (a prompt of 4096 rows: 48 % of the issue slots, 11 %
// of DRAM).  8100 rows of 32 heads take 53 us, 2.1 TB/s.  With 32 dims to a lane (E = D / 32) the sums and shuffles
// per element are fewer, but the code is longer, and a decoding step, which
// goes through it once, spends its time fetching it.  Eight dims to a lane and
// 32 (D = 128): 64 rows 6.1 and 11.2 us, 8100 rows 65 and 53 us; so prompts,
// of 32 rows and more to a sequence, take the second, unless only a part of
// their rows turns by halves (the others of its pairs are other lanes').
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256, kAppendDeep = 32;

// Rotation of a pair; every product and sum is rounded by itself, so a value
// does not depend on which of them a compiler fuses.  (Not in pairs: of two
// f32 at once the assembler fuses a product and a sum that are rounded apart.)
Q3T_DEV void turn(float &x0, float &x1, float c, float s) {
  const float y0 = x0, y1 = x1;
  x0 = __fsub_rn(__fmul_rn(y0, c), __fmul_rn(y1, s));
  x1 = __fadd_rn(__fmul_rn(y1, c), __fmul_rn(y0, s));
}
// {cos, cos, sin, sin} of the pairs f = 32 i + 8 l + e and f + 1, f even, lie in the
// order [i][e / 2][l]: neighbouring lanes read neighbouring banks
Q3T_DEV int cs_at(int f) { return (((f >> 5) << 2) + ((f >> 1) & 3)) * 4 + ((f >> 3) & 3); }

template <typename T, int D, int E>
__global__ void __launch_bounds__(kAppendThreads, E == 1 ? 4 : E == 2 ? 3 : 2) k_kv4_append(const __grid_constant__ Kv4AppendArgs a) {
  constexpr int LPR = D / 8 / E, RPW = 32 / LPR, G = D / 32, BLK = kv4_block_bytes(D), CS = D / 4 + 4;
  static_assert(E == 1 || E == G);
  extern __shared__ __align__(16) uint8_t img[];  // [kv heads of this split][BLK]
  __shared__ float4 cs[kKv4Page * CS];
  __shared__ __align__(16) float gam[2][D];
  pdl_wait();
  pdl_launch();
  Window w;
  if (!find_window(a.b, blockIdx.x, w) || w.p < 0) return;
  const int sp = a.splits, y = blockIdx.y;
  const int qh0 = (int)((int64_t)a.n_heads * y / sp), qh1 = (int)((int64_t)a.n_heads * (y + 1) / sp);
  const int kh0 = (int)((int64_t)a.c.n_kv * y / sp), kh1 = (int)((int64_t)a.c.n_kv * (y + 1) / sp);
  const int nq = qh1 - qh0, nk = kh1 - kh0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, C = lane % LPR, l = C & 3;
  const int q_items = (w.n * nq + RPW - 1) / RPW, k_items = (w.n * nk + RPW - 1) / RPW, items = q_items + 2 * k_items;
  const uint32_t inv_n = w.n == 1 ? 0u : 0xffffffffu / (uint32_t)w.n + 1u;  // divides a row's number, which is small
  // kind 0 q, 1 k, 2 v: of a warp at a time
  int kind, h, tok, item = warp, left = 0;
  int64_t ld = 0;
  const T *base = nullptr;
  auto set_kind = [&] {
    kind = item < q_items ? 0 : item < q_items + k_items ? 1 : 2;
    left = item - (kind == 0 ? 0 : kind == 1 ? q_items : q_items + k_items);
    ld = kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv;
    base = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + w.t0 * ld + (kind ? kh0 : qh0) * D + 8 * C;  // its first eight
  };
  auto fetch = [&](Raw8<T> (&x)[E]) {
    const int r = min(RPW * left + lane / LPR, w.n * (kind ? nk : nq) - 1);  // a row past the end repeats the last one
    h = w.n == 1 ? r : (int)__umulhi((uint32_t)r, inv_n);
    tok = r - h * w.n;
#pragma unroll
    for (int i = 0; i < E; i++) load8(base + tok * ld + h * D + 32 * i, a.vec, x[i]);
  };
  Raw8<T> raw[E] = {};
  set_kind();
  if (item < items) fetch(raw);
  const int page = page_of(a.c, a.b, w.s, w.p), half = a.rope.rot / 2;
  for (int i = threadIdx.x; i < w.n * half; i += kAppendThreads) {
    const int c = i / half, f = i - c * half;
    double s, co;  // angles in 64 bits: a 32-bit product is off by its position's last bits
    sincospi((double)(w.p * 16 + w.c0 + c) * a.rope.freq_pi[f], &s, &co);
    float *to = reinterpret_cast<float *>(cs + c * CS + cs_at(f)) + (f & 1);
    to[0] = (float)(co * a.rope.amplitude);
    to[2] = (float)(s * a.rope.amplitude);
  }
  for (int i = threadIdx.x; i < 2 * D; i += kAppendThreads) {
    const float *g = i < D ? a.q_gamma : a.k_gamma;
    if (g) gam[i / D][i % D] = g[i % D];
  }
  __syncthreads();
  // of the rotation by halves (E == 1), for dims 8 C .. + 3 and + 4 .. + 7: where the others of their pairs are (rot % 8 ==
  // 0, so the same element of a lane or the one four away), their sign, and the angles
  int from[2], angle[2];
  float sign[2];
  bool turns[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int d = 8 * C + 4 * e, o = d < half ? d + half : d < 2 * half ? d - half : d;
    from[e] = o >> 3;
    turns[e] = d < 2 * half;
    angle[e] = turns[e] ? cs_at(min(d, o)) : 0;
    sign[e] = d < half ? -1.f : 1.f;
  }
#pragma unroll 1
  while (item < items) {
    const int my_h = h, my_tok = tok, my_kind = kind;
    float x[E][8];
#pragma unroll
    for (int i = 0; i < E; i++) floats(raw[i], x[i]);
    item += kAppendThreads / 32;
    left += kAppendThreads / 32;
    if (item < items) {
      if (RPW * left >= w.n * (kind ? nk : nq)) set_kind();
      fetch(raw);
    }
    if (my_kind == 0 ? a.q_gamma : my_kind == 1 ? a.k_gamma : nullptr) {
      // RMSNorm.  The order of the sum leaves no trace in the 32-bit factor.
      double ss = square_sum(x);
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      const bool odd_one = !(ss > 0x1p-90 && ss < 0x1p100);  // squares outside what 32 bits hold
      if (__any_sync(0xffffffffu, odd_one)) {
        double wide = 0.0;
#pragma unroll
        for (int e = 0; e < 8 * E; e++) wide += (double)x[e >> 3][e & 7] * x[e >> 3][e & 7];
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) wide += __shfl_xor_sync(0xffffffffu, wide, d);
        ss = odd_one ? wide : ss;
      }
      const float rs = rsqrt64(ss * (1.0 / D) + (double)a.eps);
      const uint64_t r2 = f2_pack(rs, rs);
#pragma unroll
      for (int e = 0; e < 8 * E; e += 4) {
        const float4 u = *reinterpret_cast<const float4 *>(&gam[my_kind][8 * C + 32 * (e >> 3) + (e & 7)]);
        float *y = &x[e >> 3][e & 7];
        f2_split(f2_mul(f2_mul(f2_pack(y[0], y[1]), r2), f2_pack(u.x, u.y)), y[0], y[1]);
        f2_split(f2_mul(f2_mul(f2_pack(y[2], y[3]), r2), f2_pack(u.z, u.w)), y[2], y[3]);
      }
    }
    if (my_kind < 2 && half) {
      const float4 *f = cs + my_tok * CS;
      if (a.rope.interleaved) {
#pragma unroll
        for (int i = 0; i < E; i++)
          if (8 * C + 32 * i < a.rope.rot)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              const float4 u = f[cs_at(4 * C + 16 * i + (e >> 1))];
              float *y = &x[i][e];
              turn(y[0], y[1], u.x, u.z);
              turn(y[2], y[3], u.y, u.w);
            }
      } else if constexpr (E == 1) {
        float z[8];
        if (half & 4) {
#pragma unroll
          for (int e = 0; e < 8; e++) z[e] = __shfl_sync(0xffffffffu, x[0][e ^ 4], from[e >> 2], LPR);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) z[e] = __shfl_sync(0xffffffffu, x[0][e], from[0], LPR);
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float4 u = f[angle[e >> 2] + 4 * (e >> 1 & 1)];
          const float y0 = __fadd_rn(__fmul_rn(x[0][e], u.x), __fmul_rn(z[e], u.z * sign[e >> 2]));
          const float y1 = __fadd_rn(__fmul_rn(x[0][e + 1], u.y), __fmul_rn(z[e + 1], u.w * sign[e >> 2]));
          if (turns[e >> 2]) x[0][e] = y0, x[0][e + 1] = y1;
        }
      } else {  // of a whole row: both of a pair are this lane's
#pragma unroll
        for (int e = 0; e < 4 * E; e += 2) {
          float *lo = &x[e >> 3][e & 7], *hi = &x[(e >> 3) + E / 2][e & 7];
          const float4 u = f[(4 * (e >> 3) + ((e & 7) >> 1)) * 4 + l];
          turn(lo[0], hi[0], u.x, u.z);
          turn(lo[1], hi[1], u.y, u.w);
        }
      }
    }
    if (my_kind == 0) {
      __syncwarp();  // out may be q
      uint16_t *out = a.q_out + (size_t)(w.t0 + my_tok) * a.ldqo + (size_t)(qh0 + my_h) * D + 8 * C;
#pragma unroll
      for (int i = 0; i < E; i++) store8(out + 32 * i, a.vec, x[i]);
      continue;
    }
    const int c = w.c0 + my_tok, t = (c >> 1) & 3, odd = l & 1;
    uint8_t *blk = img + (size_t)my_h * BLK;
    uint32_t keys[E];
#pragma unroll
    for (int j = 0; j < E; j++) {
      const int i = E == 1 ? C >> 2 : j, ch = E == 1 ? C : 4 * j + l;  // group of 32, eight dims
      uint32_t n[8], sz;
      const uint32_t some = quantise(x[j], n, sz) ? 0xffffffffu : 0u;
      if (l == 0)
        *reinterpret_cast<uint32_t *>(blk + 16 * D + 8 * (4 * (4 * i + t) + 2 * (c >> 3) + (c & 1)) + 4 * (my_kind - 1)) = sz;
      if (my_kind == 1) {
        keys[j] = (n[0] + (n[2] << 4) + (n[4] << 8) + (n[6] << 12) + (n[1] << 16) + (n[3] << 20) + (n[5] << 24) +
                   (n[7] << 28) - kDigit * 0x11111111u) & some;
        if (E == 1) *reinterpret_cast<uint32_t *>(blk + c * (D / 2) + 4 * (G * l + i)) = keys[j];
      } else {
        // a byte has dims d and d + 8, which are this lane's and its neighbour's: each writes four
        const uint32_t first = (n[0] + (n[1] << 8) + (n[2] << 16) + (n[3] << 24) - kDigit * 0x01010101u) & some;
        const uint32_t last = (n[4] + (n[5] << 8) + (n[6] << 16) + (n[7] << 24) - kDigit * 0x01010101u) & some;
        const uint32_t theirs = __shfl_xor_sync(0xffffffffu, odd ? first : last, 1);
        const uint32_t bytes = odd ? theirs | last << 4 : first | theirs << 4;
        uint8_t *p = blk + 8 * D + 512 * (ch >> 3) + 256 * odd + 16 * t + 4 * ((ch >> 1) & 3) + 2 * (c & 1) + (c >> 3);
#pragma unroll
        for (int k = 0; k < 4; k++) p[64 * k] = (uint8_t)(bytes >> 8 * k);
      }
    }
    if (E > 1 && my_kind == 1) {
      uint8_t *p = blk + c * (D / 2) + 4 * G * l;
      if constexpr (E == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(keys[0], keys[1], keys[2], keys[3]);
      if constexpr (E == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(keys[0], keys[1]);
    }
  }
  __syncthreads();
  if (page < 0 || !nk) return;
  uint8_t *dst = a.c.pool + ((size_t)page * a.c.n_kv + kh0) * BLK;
  if (w.n == kKv4Page) {
    for (int i = threadIdx.x; i < nk * (BLK / 16); i += kAppendThreads)
      reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(img)[i];
    return;
  }
  constexpr int KW = D / 8, ITEMS = KW + G + D / 2;  // key words, scale entries, value bytes of a (token, head)
  for (int i = threadIdx.x; i < nk * w.n * ITEMS; i += kAppendThreads) {
    const int item = i % ITEMS, hc = i / ITEMS, h = hc / w.n, c = w.c0 + hc % w.n, t = (c >> 1) & 3;
    size_t at = (size_t)h * BLK;
    if (item < KW) {
      at += c * (D / 2) + 4 * item;
      *reinterpret_cast<uint32_t *>(dst + at) = *reinterpret_cast<const uint32_t *>(img + at);
    } else if (item < KW + G) {
      at += 16 * D + 8 * (4 * (4 * (item - KW) + t) + 2 * (c >> 3) + (c & 1));
      *reinterpret_cast<uint2 *>(dst + at) = *reinterpret_cast<const uint2 *>(img + at);
    } else {
      const int b = item - KW - G;  // [M][g][m]
      at += 8 * D + 512 * (b >> 5) + 64 * ((b >> 2) & 7) + 16 * t + 4 * (b & 3) + 2 * (c & 1) + (c >> 3);
      dst[at] = img[at];
    }
  }
}

// ---------------------------------------------------------------------------
// Read: one CTA per (window, head split) brings its blocks to shared memory
// and writes the rows n s + z, rounded once to bf16.  A thread takes whole
// words of digits: eight of a key, or the 64 of 16 dims of four tokens' values.
// Bound by HBM: 64 sequences of 100 to 1500 tokens, 314 MB, in 59 us, 0.81 of
// the measured copy rate (a byte at a time: 109 us).
// ---------------------------------------------------------------------------
constexpr int kReadThreads = 256;

template <int D>
__global__ void __launch_bounds__(kReadThreads) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
  constexpr int G = D / 32, BLK = kv4_block_bytes(D);
  extern __shared__ __align__(16) uint8_t img[];
  pdl_wait();
  pdl_launch();
  Window w;
  if (!find_window(a.b, blockIdx.x, w)) return;
  const int kh0 = (int)((int64_t)a.c.n_kv * blockIdx.y / a.splits);
  const int nk = (int)((int64_t)a.c.n_kv * (blockIdx.y + 1) / a.splits) - kh0;
  const int page = page_of(a.c, a.b, w.s, w.p);
  const uint4 *src = reinterpret_cast<const uint4 *>(a.c.pool + ((size_t)max(page, 0) * a.c.n_kv + kh0) * BLK);
  for (int i = threadIdx.x; i < nk * (BLK / 16); i += kReadThreads)
    cp_async16(img + 16 * i, src + i, page < 0 ? 0 : 16);  // a position that has no page reads as zeros
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  // (n s is exact in 32 bits, but may pass them where n s + z does not)
  auto value = [](uint32_t n, uint32_t sz) {
    return fmaf(__uint_as_float(0x4b000000u | n) - 0x1p23f, bf2f(sz & 0xffffu), __uint_as_float(sz & 0xffff0000u));
  };
  if (a.k)  // four threads to a row, the dims as in append
    for (int x = threadIdx.x; x < 4 * nk * w.n; x += kReadThreads) {
      const int l = x & 3, r = x >> 2, h = r / w.n, tok = r - h * w.n, c = w.c0 + tok, t = (c >> 1) & 3;
      const uint8_t *blk = img + (size_t)h * BLK;
      uint16_t *out = a.k + (size_t)(w.t0 + tok) * a.ldk + (size_t)(kh0 + h) * D + 8 * l;
      uint32_t keys[G];
      if constexpr (G == 4) {
        const uint4 u = *reinterpret_cast<const uint4 *>(blk + c * (D / 2) + 4 * G * l);
        keys[0] = u.x, keys[1] = u.y, keys[2] = u.z, keys[3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(blk + c * (D / 2) + 4 * G * l);
        keys[0] = u.x, keys[1] = u.y;
      }
#pragma unroll
      for (int i = 0; i < G; i++) {
        const uint32_t sz =
            *reinterpret_cast<const uint32_t *>(blk + 16 * D + 8 * (4 * (4 * i + t) + 2 * (c >> 3) + (c & 1)));
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = value(keys[i] >> (16 * (e & 1) + 8 * (e >> 2) + 4 * (e >> 1 & 1)) & 15u, sz);
        store8(out + 32 * i, a.vec, v);
      }
    }
  if (a.v)  // a thread has 16 dims of the four tokens that share its bytes' words
    for (int x = threadIdx.x; x < nk * (D / 4); x += kReadThreads) {
      const int m = x % (D / 16), t = x / (D / 16) & 3, h = x / (D / 4);
      const uint8_t *blk = img + (size_t)h * BLK;
      uint32_t word[8];
#pragma unroll
      for (int g = 0; g < 8; g++)
        word[g] = *reinterpret_cast<const uint32_t *>(blk + 8 * D + 512 * (m >> 2) + 64 * g + 16 * t + 4 * (m & 3));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int c = 2 * t + (j & 1) + 8 * (j >> 1), tok = c - w.c0, bit = 8 * (2 * (j & 1) + (j >> 1));
        if (tok < 0 || tok >= w.n) continue;
        const uint32_t sz = *reinterpret_cast<const uint32_t *>(blk + 16 * D + 8 * (4 * (4 * (m >> 1) + t) + j) + 4);
        uint16_t *out = a.v + (size_t)(w.t0 + tok) * a.ldv + (size_t)(kh0 + h) * D + 16 * m;
        float v[8];
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
          for (int g = 0; g < 8; g++) v[g] = value(word[g] >> (bit + 4 * n) & 15u, sz);
          store8(out + 8 * n, a.vec, v);
        }
      }
    }
}

// ---------------------------------------------------------------------------
// Attend.  With q_d the query, per group j of 32 dims
//   score = sum_j [ s_j sum_{d in j} q_d n_d + z_j sum_{d in j} q_d ]
//   out_d = sum_keys (p s_j) n_d + sum_keys p z_j,  d in group j
// so the tensor cores see digits only, and scales and zeros enter once per
// (key, group).  The digits are the A operands (16 keys x 16 dims of K, 16
// dims x 16 keys of V) and the 8 columns are (query row r, group j): column
// (r, j) of the score product holds q in the dims of group j and zeros
// elsewhere, its accumulator is the group's share of the score; column (r, j)
// of the value product holds p s_j.  (Most of the score products are with zeros;
// with few rows the tensor pipe is 24 % busy all the same.)  Every lane has work of
// its own: it scales the shares of two columns for two keys, one shuffle joins the
// groups of a row, and p s goes from the accumulator's order to the operand's
// by one matrix transpose per 8 keys.
//
// A unit is (sequence, R query rows of one kv head), R = 8 NT / G, and its
// keys go by steps of two pages; a warp streams steps through a cp.async
// ring.  Lengths are ragged, so the steps of a kv head's units are one list, cut
// into equal runs for the warps of a grid that fills the GPU once; neighbouring
// CTAs take the same run of different kv heads, whose blocks are neighbours.  A unit that
// lies inside a warp's run is finished there; the (m, l, o) parts of one that
// does not are joined in order, by the CTA where it has them all, otherwise
// by k_kv4_combine from the workspace.  Nothing is kept between calls.
//
// Long caches are bound by HBM: 64 requests of 4096 keys on 8 kv heads, 336
// MB, take 65 us, 0.79 of the measured copy rate; one of 131071 keys 37 us (in
// units of CTAs that end with a sequence 94).  Short ones are bound by both ends,
// filling the ring and joining the parts: 64 of 100 to 1500 keys 26 us.
//
// f16 holds q times a power of two per row (its 11 bits keep a bf16 q whole
// down to 2^-25 of the row's largest) and p s, which is rounded to 11 bits, as
// against the 8 of the output.  p is taken from a reference that follows the
// largest weight times scale that a row has seen, not the largest scale: p s is
// at most 2^15, and 2^10 where the reference moves, so it has all its bits down
// to 2^-24 of the row's largest, and values that have no weight, or that the row
// may not see, cost the others nothing.  l and o carry the reference too, and it
// leaves with the division.  All sums, references and l are in 32 bits.
// ---------------------------------------------------------------------------
Q3T_DEV void mma_f16(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
Q3T_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
Q3T_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
Q3T_DEV float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(14 - exponent of x), so that x times it lies in [2^14, 2^15)
Q3T_DEV float to_2p14(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 0xff);  // x >= 0
  const int f = min(max(127 + 14 + 127 - e, 1), 253);
  return __uint_as_float((uint32_t)f << 23);
}
// exponent of x >= 0 as a float's field has it
Q3T_DEV int exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }
// an 8 x 8 tile of f16, rows in accumulator order, transposed
Q3T_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// A part's l lies in [2^kPartL, 2^(kPartL + 1)): with it o is so far below the values that neither the largest ones nor
// the sum of a thousand parts leave 32 bits.
constexpr int kPartL = -11;
// weight of a part with running maximum m and sum l under the joint maximum
// M; a part without keys has none, one with NaN scores keeps them
Q3T_DEV float part_weight(float m, float l, float M) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return ex2(m - M);
}

// A sequence's rows, as the kernel keeps them: token rows from t0, n * heads
// of a kv head = `total` query rows, the first at position pos0.
struct SeqRows {
  int t0, total, pos0, table_row, row0;  // row0: of the unit
};
// Query rows [row0, row0 + nrow) of it and the pages they see.
struct Unit {
  int row0, nrow, pos_lo, pos_hi, pg_lo, pages;
};
// token of a query row: a decode step has one, and no division then
Q3T_DEV int token_of(int row, int gq) { return row < gq ? 0 : row / gq; }
// the first key that the row at `pos` sees: a difference only where it does not pass 0, as `pos` may be far below it and
// `window` near the largest number
Q3T_DEV int first_key(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }
template <int R>
Q3T_DEV Unit unit_of(const SeqRows &s, int row0, int gq, int window, int table_stride) {
  Unit u;
  u.row0 = row0;
  u.nrow = min(R, s.total - row0);
  u.pos_lo = s.pos0 + token_of(row0, gq);
  u.pos_hi = s.pos0 + token_of(row0 + max(u.nrow, 1) - 1, gq);
  u.pg_lo = first_key(u.pos_lo, window) >> 4;
  u.pages = u.pos_hi < 0 ? 0 : max(0, min((u.pos_hi >> 4) + 1, table_stride) - u.pg_lo);  // none past the table
  return u;
}
// steps of a unit: one at least, so that rows without keys are answered too
constexpr int kStepPages = 2, kFoldSteps = 16;
Q3T_DEV int unit_steps(const Unit &u) { return u.nrow > 0 ? max(1, (u.pages + kStepPages - 1) / kStepPages) : 0; }

template <int D, int NT>
struct AttendCfg {
  static constexpr int G = D / 32, R = NT * 8 / G, BLK = kv4_block_bytes(D);
  static constexpr int NP = kStepPages, ST = 2;  // pages of a step, steps in the ring
  static constexpr int W = 4;                    // warps of a CTA
  static constexpr int RING = ST * NP * BLK;
  static constexpr int PART = R * (2 + G + D);   // floats of a part: m [R], l [R], z [R][G], o [R][D]
  static constexpr int MAXSEQ = 512;             // units of a launch's list
  static constexpr size_t smem(int units) {
    return (size_t)W * RING + W * 2 * PART * 4 + units * sizeof(SeqRows) + (units + 1) * 4;
  }
};

template <int D>
Q3T_DEV void store_out(const Kv4AttendArgs &a, int t0, int row, int kvh, int d, float L, float o) {
  const int gq = a.n_heads / a.c.n_kv, tok = token_of(row, gq), head = kvh * gq + row - tok * gq;
  a.out[(size_t)(t0 + tok) * a.ldo + (size_t)head * D + d] = f2bf(L == 0.f ? 0.f : o / L);  // no keys: zeros
}

// The step list of a kv head: steps pre[i] .. pre[i + 1] - 1 are those of
// rows [seq[i].row0, seq[i].row0 + R) of a sequence.
struct StepList {
  const int *pre;
  const SeqRows *seq;
  int n;
};

// Where the copies of a warp's run are: the block of up to 16 steps of one
// unit whose pages are in `ids` (by lane), and the block after it.
template <int R>
struct PageCursor {
  int seq, step, end;   // sequence, next step of its unit, end of the unit's steps in the run
  int block, left;      // first step of the block, steps of the run not yet taken
  int pg_lo, pages;     // of the unit
  int ids, next_ids;
  int next_seq, next_step, next_end, next_lo, next_pages;
  static constexpr int kBlock = 32 / kStepPages;

  Q3T_DEV void look(const Kv4AttendArgs &a, const StepList &L, int s, int step, int lo, int n, int &out) {
    const int p = lo + step * kStepPages + (threadIdx.x & 31);
    out = -1;
    if (p < lo + n && p < a.c.table_stride) {
      const int row = L.seq[s].table_row;
      if (row >= 0 && row < a.c.table_rows) out = a.c.table[(size_t)row * a.c.table_stride + p];
    }
  }
  // the block after (seq, block), its pages on their way
  Q3T_DEV void after(const Kv4AttendArgs &a, const StepList &L, int gq, int left_after) {
    next_seq = seq, next_step = block + kBlock, next_end = end, next_lo = pg_lo, next_pages = pages;
    if (next_step >= end) {
      if (left_after <= 0) {
        next_ids = -1;
        return;
      }
      next_step = 0;
      do next_seq++;
      while (L.pre[next_seq + 1] == L.pre[next_seq]);
      next_end = min(L.pre[next_seq + 1] - L.pre[next_seq], left_after);
      const Unit u = unit_of<R>(L.seq[next_seq], L.seq[next_seq].row0, gq, a.window, a.c.table_stride);
      next_lo = u.pg_lo, next_pages = u.pages;
    }
    look(a, L, next_seq, next_step, next_lo, next_pages, next_ids);
  }
  Q3T_DEV void start(const Kv4AttendArgs &a, const StepList &L, int gq, int s, int at, int to) {
    const Unit u = unit_of<R>(L.seq[s], L.seq[s].row0, gq, a.window, a.c.table_stride);
    seq = s, step = block = at - L.pre[s], left = to - at;
    end = min(L.pre[s + 1] - L.pre[s], step + left);
    pg_lo = u.pg_lo, pages = u.pages;
    look(a, L, s, step, pg_lo, pages, ids);
  }
  // one step taken (after() once before the first)
  Q3T_DEV void advance(const Kv4AttendArgs &a, const StepList &L, int gq) {
    step++, left = max(left - 1, 0);
    if (left > 0 && (step == end || step == block + kBlock)) {
      seq = next_seq, step = block = next_step, end = next_end, pg_lo = next_lo, pages = next_pages, ids = next_ids;
      after(a, L, gq, left - (end - step));
    }
  }
};

// What became of a warp's run: up to two parts that are not a whole unit.
struct RunSlot {
  int seq, begins, ends;  // -1: none
};

// Steps [at, to) of kv head kvh's list, by one warp.  Units that lie inside
// are written out, parts of others go to part[0] and part[1].
template <int D, int NT>
Q3T_DEV void attend_run(const Kv4AttendArgs &a, const StepList &L, int kvh, int at, int to, uint8_t *ring,
                        float *part_base, RunSlot *slot) {
  using Cfg = AttendCfg<D, NT>;
  constexpr int G = Cfg::G, R = Cfg::R, BLK = Cfg::BLK, NP = Cfg::NP, ST = Cfg::ST, MT = D / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, j = g % G, gq = a.n_heads / a.c.n_kv;
  if (lane < 2) slot[lane].seq = -1;
  if (at >= to) return;
  int seq;
  {
    int lo = 0, hi = L.n;  // the last sequence whose steps begin at or before `at`: it has some
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.pre[mid] <= at)
        lo = mid;
      else
        hi = mid;
    }
    seq = lo;
  }

  // bf16 queries of a sequence's unit: column g, dims 32 j + 8 t .. + 7
  auto load_q = [&](int s, uint32_t (&x)[NT][4]) {
    const SeqRows sq = L.seq[s];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int flat = min(sq.row0 + (nt * 8 + g) / G, sq.total - 1);  // a row past the end repeats the last one
      const int tok = token_of(flat, gq), head = kvh * gq + flat - tok * gq;
      const uint16_t *qp = a.q + (size_t)(sq.t0 + tok) * a.ldq + (size_t)head * D + 32 * j + 8 * t;
      if (a.vec) {
        const uint4 w = *reinterpret_cast<const uint4 *>(qp);
        x[nt][0] = w.x, x[nt][1] = w.y, x[nt][2] = w.z, x[nt][3] = w.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[nt][i] = qp[2 * i] | (uint32_t)qp[2 * i + 1] << 16;
      }
    }
  };
  uint32_t raw_q[NT][4];  // of the next unit
  load_q(seq, raw_q);

  // ---- ring ----
  PageCursor<R> cur;
  cur.start(a, L, gq, seq, at, to);
  uint32_t has = 0;  // whether a page is there, the newest step in the low bits
  int put = 0;       // the stage of the next copies
  const uint8_t *pool = a.c.pool + (size_t)kvh * BLK + 16 * lane;
  auto copies = [&] {
    has <<= NP;
    if (cur.left > 0) {
      uint8_t *dst = ring + put * (NP * BLK) + 16 * lane;
#pragma unroll
      for (int k = 0; k < NP; k++) {
        const int id = __shfl_sync(0xffffffffu, cur.ids, (cur.step - cur.block) * NP + k);
        if (id >= 0 && id < a.c.num_pages) {
          has |= 1u << k;
          const uint8_t *src = pool + (size_t)id * a.c.n_kv * BLK;
#pragma unroll
          for (int i = 0; i < (BLK / 16 + 31) / 32; i++)
            if (BLK % 512 == 0 || lane + 32 * i < BLK / 16) cp_async16(dst + k * BLK + 512 * i, src + 512 * i, 16);
        }
      }
      put = put + 1 == ST ? 0 : put + 1;
    }
    cp_async_commit();
  };
  copies();
  cur.after(a, L, gq, cur.left - (cur.end - cur.step));
  cur.advance(a, L, gq);
#pragma unroll
  for (int i = 1; i < ST - 1; i++) {
    copies();
    cur.advance(a, L, gq);
  }
  int get = 0, parts = 0;
  while (at < to) {
    const SeqRows sq = L.seq[seq];
    const Unit u = unit_of<R>(sq, sq.row0, gq, a.window, a.c.table_stride);
    const int steps = L.pre[seq + 1] - L.pre[seq], i0 = at - L.pre[seq], i1 = min(steps, i0 + (to - at));
    const int pos_lo = u.pos_lo, pos_hi = u.pos_hi;

    // ---- queries ----
    uint32_t qb[NT][G][2][2];  // zeros outside group j
    float qs[NT][2], sc[NT];   // accumulator order: of columns 2 t and 2 t + 1, of their row
    int lim[NT], low[NT];      // the keys that row sees
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; i++)
        v[2 * i] = bf2f(raw_q[nt][i] & 0xffffu), v[2 * i + 1] = __uint_as_float(raw_q[nt][i] & 0xffff0000u);
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[i])), sum += v[i];
#pragma unroll
      for (int o = 1; o < 4 * G; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // a negative scale turns the queries and a scale of zero clears them, so
      // that below sc > 0 and the largest x is the largest score
      const float f = a.scale == 0.f ? 0.f : a.scale < 0.f ? -to_2p14(top) : to_2p14(top);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= f;
      // dims 0, 1 meet digits n 2^-24, dims 2, 3 meet 16 n 2^-24
      const uint32_t q4[4] = {pack_f16x2(v[0], v[1]), pack_f16x2(v[2] * 0.0625f, v[3] * 0.0625f), pack_f16x2(v[4], v[5]),
                              pack_f16x2(v[6] * 0.0625f, v[7] * 0.0625f)};
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int i = 0; i < 4; i++) qb[nt][q][i >> 1][i & 1] = q == j ? q4[i] : 0u;
      sum *= f * 0x1p-24f;
      qs[nt][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
      qs[nt][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      // (2^24 where it can neither pass 32 bits nor vanish before its time; never 0, as -inf times it has to stay that)
      const float back = f < 1.f && f > -1.f ? a.scale / f * 0x1p24f : a.scale * (0x1p24f / f);
      sc[nt] = __shfl_sync(0xffffffffu, a.scale == 0.f ? 1.f : fminf(fmaxf(back, FLT_MIN), FLT_MAX), 8 * t);
      lim[nt] = sq.pos0 + token_of(min(u.row0 + (nt * 8 + 2 * t) / G, sq.total - 1), gq);
      low[nt] = first_key(lim[nt], a.window);
    }
    int next = seq;  // the unit after this one, its queries on their way
    if (i1 - i0 < to - at) {
      do next++;
      while (L.pre[next + 1] == L.pre[next]);
      load_q(next, raw_q);
    }

    // p = 2^(x sc - mu), mu = ref where a key has been seen and 0 before: ref follows the largest weight times size,
    // x sc + log2 of a key's size, so that p s is up to 2^15
    float ref[NT], mu[NT], l[NT], zac[NT][2], acc[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      ref[nt] = -INFINITY;
      mu[nt] = 0.f;
      l[nt] = zac[nt][0] = zac[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; i++) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
    }

    for (int it = i0; it < i1; it++) {
      copies();
      cur.advance(a, L, gq);
      cp_async_wait<ST - 1>();
      __syncwarp();
      const int p0 = u.pg_lo + it * NP;
      const uint8_t *blk0 = ring + get * (NP * BLK);
      get = get + 1 == ST ? 0 : get + 1;
      const uint32_t here = has >> ((ST - 1) * NP);  // bit k: page k of this step
      // ---- digits of q . k, then x[nt][k][h]: key g + 8 h of page k ----
      float x[NT][NP][2];
      uint32_t vz[NP][2][2];  // value scale and zero of key g + 8 h, groups of columns 2 t and 2 t + 1
#pragma unroll
      for (int k = 0; k < NP; k++) {
        const uint8_t *blk = blk0 + k * BLK;
        uint32_t kw[2][G];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (G == 4) {
            const uint4 w = *reinterpret_cast<const uint4 *>(blk + 16 * lane + 512 * h);
            kw[h][0] = w.x, kw[h][1] = w.y, kw[h][G - 2] = w.z, kw[h][G - 1] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(blk + 8 * lane + 256 * h);
            kw[h][0] = w.x, kw[h][1] = w.y;
          }
        }
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
        for (int q = 0; q < G; q++)
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const uint32_t y0 = kw[0][q] >> 8 * b, y1 = kw[1][q] >> 8 * b;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              mma_f16(c[nt], y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qb[nt][q][b][0],
                      qb[nt][q][b][1]);
          }
        const uint8_t *kp = blk + 16 * D + 128 * (2 * t % G) + 32 * (g >> 1) + 8 * (g & 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint2 s0 = *reinterpret_cast<const uint2 *>(kp + 16 * h);
          const uint2 s1 = *reinterpret_cast<const uint2 *>(kp + 16 * h + 128);
          vz[k][h][0] = s0.y;
          vz[k][h][1] = s1.y;
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            float y = __uint_as_float(s0.x & 0xffff0000u) * qs[nt][0];
            y = fmaf(__uint_as_float(s1.x & 0xffff0000u), qs[nt][1], y);
            y = fmaf(bf2f(s0.x & 0xffffu), c[nt][2 * h], y);
            y = fmaf(bf2f(s1.x & 0xffffu), c[nt][2 * h + 1], y);
            if (G == 4) y += __shfl_xor_sync(0xffffffffu, y, 1);
            x[nt][k][h] = y;
          }
        }
        // keys that a row may not see, and pages that are not there: whatever
        // the slot holds, scales that are no numbers included, does not count
        const bool there = here >> k & 1;
        const int key0 = (p0 + k) * 16;
        if (!there || key0 + 15 > pos_lo || key0 < first_key(pos_hi, a.window)) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int key = key0 + g + 8 * h;
            bool any = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const bool seen = there && key <= lim[nt] && key >= low[nt];
              if (!seen) x[nt][k][h] = -INFINITY;
              any |= seen;
            }
            if (!any) vz[k][h][0] = vz[k][h][1] = 0u;
          }
        }
      }
      // ---- largest weight times size ----
      float top[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) top[nt] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2 * NP; i++) {
        // A key's size is its largest scale.  Zeros count too, from 2^20 times that on, so that p times them stays in 32
        // bits, and so do sizes below 2^-86, for p's own sake.
        const uint32_t v0 = vz[i >> 1][i & 1][0], v1 = vz[i >> 1][i & 1][1];
        const float zero = fmaxf(fabsf(__uint_as_float(v0 & 0xffff0000u)), fabsf(__uint_as_float(v1 & 0xffff0000u)));
        const float size = fmaxf(fmaxf(bf2f(v0 & 0xffffu), bf2f(v1 & 0xffffu)), fmaxf(zero * 0x1p-20f, 0x1p-86f));
        const float e = lg2(size);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) top[nt] = fmaxf(top[nt], fmaf(x[nt][i >> 1][i & 1], sc[nt], e));
      }
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) moved |= top[nt] > ref[nt] + 15.f;
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
          for (int o = G == 4 ? 1 : 4; o < 32; o = o == 1 ? 4 : 2 * o)  // over a row's keys, and its lanes' groups
            top[nt] = fmaxf(top[nt], __shfl_xor_sync(0xffffffffu, top[nt], o));
          if (top[nt] > ref[nt] + 15.f) {  // the first time, or past what p s is to hold
            const float to = top[nt] - 10.f, f = ref[nt] == -INFINITY ? 0.f : ex2(ref[nt] - to);
            ref[nt] = mu[nt] = to;
            l[nt] *= f;
            zac[nt][0] *= f;
            zac[nt][1] *= f;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
              for (int e = 0; e < 4; e++) acc[nt][i][e] *= f;
          }
        }
      }
      // ---- p, p s and the value product ----
#pragma unroll
      for (int k = 0; k < NP; k++) {
        const uint8_t *blk = blk0 + k * BLK;
        uint32_t b[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const float p = ex2(fmaf(x[nt][k][h], sc[nt], -mu[nt]));
            l[nt] += p;
            // a key that only another row of this lane sees: its value may be anything
            const bool out = NT > 1 && x[nt][k][h] == -INFINITY;
            float w[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              w[e] = out ? 0.f : p * bf2f(vz[k][h][e] & 0xffffu);
              zac[nt][e] = out ? zac[nt][e] : fmaf(p, __uint_as_float(vz[k][h][e] & 0xffff0000u), zac[nt][e]);
            }
            b[nt][h] = transpose8(pack_f16x2(w[0], w[1]));
          }
#pragma unroll
        for (int M = 0; M < D / 64; M++) {
          const uint4 w = *reinterpret_cast<const uint4 *>(blk + 8 * D + 512 * M + 16 * lane);
          const uint32_t v4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t v = v4[i], v8 = v >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              mma_f16(acc[nt][4 * M + i], v & 0x000f000fu, v & 0x00f000f0u, v8 & 0x000f000fu, v8 & 0x00f000f0u, b[nt][0],
                      b[nt][1]);
          }
        }
      }
      __syncwarp();  // every lane is done with the stage that the next copies write
      if (it % kFoldSteps == kFoldSteps - 1) {
        // Digits are 0..15, so their sums grow with the keys and the zeros' take most of it off again: what 25000 keys
        // round away was 3 % of their average.  Taken off in time, a sum stays as small as its result.
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float z = zac[nt][e];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
            zac[nt][e] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; i++) {
              acc[nt][i][e] = fmaf(z, 0x1p-24f, acc[nt][i][e]);
              acc[nt][i][2 + e] = fmaf(z, 0x1p-20f, acc[nt][i][2 + e]);
            }
          }
      }
    }
    float *part = part_base + parts * Cfg::PART;
    float *p_m = part, *p_l = p_m + R, *p_z = p_l + R, *p_o = p_z + R * G;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], o);
        zac[nt][0] += __shfl_xor_sync(0xffffffffu, zac[nt][0], o);
        zac[nt][1] += __shfl_xor_sync(0xffffffffu, zac[nt][1], o);
      }
      const int r = (nt * 8 + 2 * t) / G, ja = 2 * t % G;
      // l as a number of kPartL and an exponent, which ref takes: refs may be so far apart that one of two parts of like
      // weight would have none.  (0 and no number stay that.)
      const int el = l[nt] == 0.f ? 0 : min(max(exponent(l[nt]) - kPartL, -126), 126);
      const float fl = __uint_as_float((uint32_t)(127 - el) << 23);
      if (g == 0) {
        p_z[r * G + ja] = zac[nt][0] * fl;
        p_z[r * G + ja + 1] = zac[nt][1] * fl;
        if (ja == 0) {
          p_m[r] = ref[nt] + (float)el;
          p_l[r] = l[nt] * fl;
        }
      }
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (ja + e == i / 2) {  // digits were n 2^-24 and 16 n 2^-24
            p_o[r * D + 16 * i + g] = acc[nt][i][e] * 0x1p24f * fl;
            p_o[r * D + 16 * i + 8 + g] = acc[nt][i][2 + e] * 0x1p20f * fl;
          }
    }
    __syncwarp();
    if (i0 == 0 && i1 == steps) {
      for (int e = lane; e < u.nrow * D; e += 32)
        store_out<D>(a, sq.t0, u.row0 + e / D, kvh, e % D, p_l[e / D], p_o[e] + p_z[e / 32]);
      __syncwarp();
    } else {
      if (lane == 0) slot[parts] = RunSlot{seq, i0 == 0, i1 == steps};
      parts++;
    }
    at += i1 - i0;
    seq = next;
  }
  cp_async_wait<0>();
  __syncwarp();
}

// What a CTA says of the unit that begins in its run and goes on in others:
// n CTAs have parts of it (0: there is none), and where its rows are.
struct PartNote {
  int n, t0, row0, nrow;
};
// Workspace: notes [CTAs], parts [CTAs][2][PART]; CTA c works on kv head
// c % n_kv, and c + n_kv goes on where it ends.  Part 0 belongs to a unit that
// began in an earlier CTA, part 1 to one that begins here and goes on.

// The steps of list L of kv head kvh that CTA ci of `ctas` has, and what is left of them.
template <int D, int NT>
Q3T_DEV void attend_list(const Kv4AttendArgs &a, const StepList &L, int kvh, int ci, int ctas, uint8_t *ring_all,
                         float *s_part, RunSlot (*slot)[2], PartNote *note, float *parts) {
  using Cfg = AttendCfg<D, NT>;
  constexpr int R = Cfg::R, W = Cfg::W, PART = Cfg::PART;
  const int warp = threadIdx.x >> 5;
  const int64_t T = L.pre[L.n], runs = (int64_t)ctas * W, run = (int64_t)ci * W + warp;
  attend_run<D, NT>(a, L, kvh, (int)(T * run / runs), (int)(T * (run + 1) / runs), ring_all + warp * Cfg::RING,
                    s_part + warp * 2 * PART, slot[warp]);
  __syncthreads();
  PartNote left{0, 0, 0, 0};
  // units that more than one run of this CTA, or of others, has parts of
  int owner[2 * W];
#pragma unroll
  for (int k = 0; k < 2 * W; k++) owner[k] = slot[k >> 1][k & 1].seq;
  uint32_t left_to_join = 0;
#pragma unroll
  for (int k = 0; k < 2 * W; k++) left_to_join |= (owner[k] >= 0 ? 1u : 0u) << k;
  while (left_to_join) {
    const int first = __ffs(left_to_join) - 1;
    const RunSlot f = slot[first >> 1][first & 1];
    uint32_t mine = 0;  // its parts: the next ones of the same sequence
#pragma unroll
    for (int k = 0; k < 2 * W; k++) mine |= (owner[k] == f.seq ? 1u : 0u) << k;
    left_to_join &= ~mine;
    const int last = 31 - __clz(mine), ends = slot[last >> 1][last & 1].ends;
    const SeqRows sq = L.seq[f.seq];
    const int nrow = min(R, sq.total - sq.row0);
    float *dst = parts + (f.begins ? PART : 0);
#pragma unroll
    for (int e0 = 0; e0 < R * D; e0 += 128) {
      const int e = e0 + threadIdx.x, r = e / D, d = e - r * D;
      float M = -INFINITY, l = 0.f, o = 0.f, pm[2 * W];
#pragma unroll
      for (int k = 0; k < 2 * W; k++) {
        pm[k] = mine >> k & 1 ? s_part[k * PART + r] : -INFINITY;
        M = fmaxf(M, pm[k]);
      }
#pragma unroll
      for (int k = 0; k < 2 * W; k++) {
        if (!(mine >> k & 1)) continue;
        const float *p = s_part + k * PART;
        const float w = part_weight(pm[k], p[R + r], M);
        l += w * p[R + r];
        o += w * (p[2 * R + R * Cfg::G + e] + p[2 * R + e / 32]);
      }
      if (f.begins && ends) {
        if (r < nrow) store_out<D>(a, sq.t0, sq.row0 + r, kvh, d, l, o);
      } else {
        dst[2 * R + R * Cfg::G + e] = o;  // with its zeros
        if (d == 0) {
          dst[r] = M;
          dst[R + r] = l;
        }
      }
    }
    if (f.begins && !ends) {
      const int64_t e = L.pre[f.seq + 1] - 1;  // the unit's last step, and the CTA that has it
      int c = (int)(e * ctas / T);
      while (c + 1 < ctas && T * (c + 1) / ctas <= e) c++;
      left = PartNote{c - ci + 1, sq.t0, sq.row0, nrow};
    }
  }
  if (ctas > 1) {
    if (threadIdx.x == 0) *note = left;
    if (T * ci / ctas == T * (ci + 1) / ctas && threadIdx.x < R) {  // no steps: a part that weighs nothing
      parts[threadIdx.x] = -INFINITY;
      parts[R + threadIdx.x] = 0.f;
    }
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(128, NT == 1 ? 3 : 2) k_kv4_attend(const __grid_constant__ Kv4AttendArgs a,
                                                                     PartNote *notes, float *parts) {
  using Cfg = AttendCfg<D, NT>;
  constexpr int R = Cfg::R, W = Cfg::W, PART = Cfg::PART;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ int warp_tot[W], one_pre[2];
  __shared__ SeqRows one_seq;
  __shared__ RunSlot slot[W][2];
  const int B = a.b.num_seqs, U = a.units, E = B * U, n_kv = a.c.n_kv, gq = a.n_heads / n_kv;
  float *s_part = reinterpret_cast<float *>(ring_all + W * Cfg::RING);   // [W][2][PART]
  SeqRows *seq = reinterpret_cast<SeqRows *>(s_part + W * 2 * PART);     // [E], a sequence's U units in turn
  int *pre = reinterpret_cast<int *>(seq + E);                           // [E + 1]
  pdl_wait();
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int carry = 0, more = 0;
  for (int base = 0; notes && base < E; base += 128) {
    const int e = base + (int)threadIdx.x;
    int incl = 0;
    if (e < E) {
      const int s = e / U;
      SeqRows q;
      int n;
      seq_rows(a.b, s, q.t0, n, q.pos0);
      q.total = n * gq;
      q.table_row = a.b.table_row ? a.b.table_row[s] : a.b.first + s;
      q.row0 = (e - s * U) * R;
      if (a.big > 0 && q.total > a.big) q.total = 0;  // k_kv4_prompt has it
      seq[e] = q;
      incl = unit_steps(unit_of<R>(q, q.row0, gq, a.window, a.c.table_stride));
      more |= q.total > U * R;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int k = 0; k < W; k++) {
      if (k < warp) before += warp_tot[k];
      carry += warp_tot[k];
    }
    if (e < E) pre[e + 1] = before + incl;
    __syncthreads();
  }
  if (notes && threadIdx.x == 0) pre[0] = 0;
  more = __syncthreads_or(more);
  // attend_list is here once: its code, twice or three times, would be fetched more than run
  for (int turn = 0;; turn++) {
    StepList list{pre, seq, E};
    int kvh = blockIdx.x % n_kv, ci = blockIdx.x / n_kv, ctas = gridDim.x / n_kv;
    if (!notes || turn > 0) {
      int s, i;
      if (!notes) {  // a CTA to each unit
        s = ci / U, i = ci - s * U + turn * U;
        if (threadIdx.x == 0) {
          int n;
          seq_rows(a.b, s, one_seq.t0, n, one_seq.pos0);
          one_seq.total = a.big > 0 && n * gq > a.big ? 0 : n * gq;
          one_seq.table_row = a.b.table_row ? a.b.table_row[s] : a.b.first + s;
        }
      } else {  // rows beyond a sequence's U units (more than the caller announced): a CTA to each R of them
        if (!more || !find_item(B, blockIdx.x + (turn - 1) * gridDim.x,
                                [&](int q) { return max(0, (seq[q * U].total + R - 1) / R - U) * n_kv; }, s, i))
          break;
        kvh = i % n_kv, i = i / n_kv + U;
        if (threadIdx.x == 0) one_seq = seq[s * U];
      }
      if (threadIdx.x == 0) {
        one_seq.row0 = i * R;
        one_pre[0] = 0;
        one_pre[1] = unit_steps(unit_of<R>(one_seq, i * R, gq, a.window, a.c.table_stride));
      }
      __syncthreads();
      if (i * R >= one_seq.total) break;
      list = StepList{one_pre, &one_seq, 1};
      ci = 0, ctas = 1;
    }
    attend_list<D, NT>(a, list, kvh, ci, ctas, ring_all, s_part, slot, notes ? notes + blockIdx.x : nullptr,
                       parts + (size_t)blockIdx.x * 2 * PART);
    __syncthreads();
  }
}

// Joins the units whose parts several CTAs left: CTA b takes the one that
// begins in CTA b of the attend launch, its warps a part each in turn, so that
// the loads of a few parts are one latency and those of many are spread.
template <int D, int NT>
__global__ void __launch_bounds__(256) k_kv4_combine(const __grid_constant__ Kv4AttendArgs a, const PartNote *notes,
                                                     const float *parts) {
  using Cfg = AttendCfg<D, NT>;
  constexpr int R = Cfg::R, G = Cfg::G, PART = Cfg::PART, PER = R * D / 32, WARPS = 8;
  __shared__ float s_m[WARPS][R], s_l[WARPS][R], s_o[WARPS][R * D];
  pdl_wait();
  pdl_launch();
  const int n_kv = a.c.n_kv, b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PartNote f = notes[b];
  if (f.n == 0) return;
  // lane's elements are lane + 32 i of row (32 i) / D
  float m[R], l[R], o[PER];
#pragma unroll
  for (int r = 0; r < R; r++) m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
  for (int i = 0; i < PER; i++) o[i] = 0.f;
  constexpr int BATCH = 4;  // parts whose loads are in flight together
  for (int k0 = warp; k0 < f.n; k0 += WARPS * BATCH) {
    float pm[BATCH][R], pl[BATCH][R], po[BATCH][PER];
#pragma unroll
    for (int x = 0; x < BATCH; x++) {
      const int k = k0 + x * WARPS;
      const float *p = parts + ((size_t)(b + k * n_kv) * 2 + (k == 0 ? 1 : 0)) * PART;
#pragma unroll
      for (int r = 0; r < R; r++) pm[x][r] = k < f.n ? p[r] : -INFINITY, pl[x][r] = k < f.n ? p[R + r] : 0.f;
#pragma unroll
      for (int i = 0; i < PER; i++) po[x][i] = k < f.n ? p[2 * R + R * G + lane + 32 * i] : 0.f;
    }
#pragma unroll
    for (int x = 0; x < BATCH; x++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float M = fmaxf(m[r], pm[x][r]), f0 = part_weight(m[r], l[r], M), f1 = part_weight(pm[x][r], pl[x][r], M);
        m[r] = M;
        l[r] = f0 * l[r] + f1 * pl[x][r];
#pragma unroll
        for (int i = r * (D / 32); i < (r + 1) * (D / 32); i++)  // what weighs nothing may be anything
          o[i] = (f0 == 0.f ? 0.f : f0 * o[i]) + (f1 == 0.f ? 0.f : f1 * po[x][i]);
      }
  }
  if (lane == 0)
#pragma unroll
    for (int r = 0; r < R; r++) s_m[warp][r] = m[r], s_l[warp][r] = l[r];
#pragma unroll
  for (int i = 0; i < PER; i++) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  for (int e = threadIdx.x; e < f.nrow * D; e += 256) {
    const int r = e / D, d = e - r * D;
    float M = -INFINITY, L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) M = fmaxf(M, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f1 = part_weight(s_m[w][r], s_l[w][r], M);
      L += f1 * s_l[w][r];
      x += f1 * s_o[w][e];
    }
    store_out<D>(a, f.t0, f.row0 + r, b % n_kv, d, L, x);
  }
}

// ---------------------------------------------------------------------------
// Attend for many rows: a prompt or a chunk of one.  128 query rows (tokens x
// heads of a kv head) are one tile of tcgen05 products, so a block is unpacked
// once for many rows, to f16 in the swizzled order the tensor core reads:
//   S = Q K^T     M 128 rows, N 64 keys, K D        (TMEM, two buffers)
//   O += P V      M 128 rows, N D, K 64 keys        (TMEM)
// Two such halves share every unpacked tile of keys.  Warps 0-7 are the
// softmax (a thread to a row), 8-15 unpack (a warp to a page of K or of V of
// the tile), 16-19 issue the products, one lane to each half's S and P V (with
// one for both halves' S and one for both P V a prompt took 9 us more).  K, V and S
// have two buffers each, so the unpacking of a tile, its S, the softmax of the
// one before and its P V run at once.
//
// What bounds it is the softmax warps' way through a tile: waits for S, V and
// TMEM loads, 64 exponentials a row, and a share of the schedulers, whose slots
// are 59 % taken, by the unpacking warps too (which 4-bit keys cost and bf16 ones
// would not).  The tensor pipe is busy 23 %, HBM 2 %.  A prompt of 4096 tokens on
// 8 kv heads (68.7 GFLOP) takes 120 us, 0.35 of the products' rate alone.  With
// loops unrolled throughout, 102 KB of code instead of 62, warps waited for
// instructions most of the time: 178 us.  One buffer of P, whose P V a softmax
// then waits for, is 5 us more; powers of two that follow the weights, and keys'
// own, 3.4 us (a page's alone are wrong beside a large value without weight).
//
// Where tiles of rows cannot fill the GPU, CTAs share the keys of each and
// k_kv4_join joins their parts: 32 rows of one request on 8000 keys, 126 tiles,
// take 30 us.
//
// f16 holds q times a power of two per row, K and V times one per page (from the
// largest value there, 11 bits of each), or per key where a page has keys of less
// than 2^-10 of its largest.  K's power enters with the score's scale, V's with p: P of a key is 2^(score + V's power - ref),
// and l sums it without V's power.  So ref follows the largest weight times value
// that a row sees, not the largest value: one that has no weight takes no bits of
// the others, nor does one that the row may not see.  l, S and O are in 32 bits;
// ref is moved, and O with it, only when P would pass 2^15, and then to a P of 2^7,
// so that P has all its bits from 2^-14 to there.  (Dims below 2^-28 of their
// key's largest lose bits.)
//
// What a row may not see must not touch it: K and V of keys that no row of the
// tile sees are zeros, and a group that is no number becomes zeros too and is
// noted, so that the rows that do see it, and no others, come out as NaN.
// ---------------------------------------------------------------------------
Q3T_DEV void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// whether the barrier's phase `parity` is complete, after some time of waiting for it
Q3T_DEV bool mbar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// 32 TMEM lanes x 32 consecutive columns; call tmem_wait_ld() before reading r
Q3T_DEV void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
Q3T_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
Q3T_DEV uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Eight digits of a word as four f16 pairs n s + z: 0x6400 | n is 1024 + n,
// 0x6400 | 16 n is 1024 + 16 n.  Taken as the subnormals they are, digits cost
// half the instructions but leave s only 2^-24 of f16's range: a key far below
// the largest of its page would lose its bits.
Q3T_DEV void unpack8(uint32_t w, const uint32_t s[2], const uint32_t z[2], uint32_t out[4]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t x = i ? w >> 8 : w;
    const uint32_t lo = h2_fma((x & 0x000f000fu) | 0x64006400u, 0x3c003c00u, 0xe400e400u);  // - 1024
    const uint32_t hi = h2_fma((x & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd400d400u);  // / 16 - 64
    out[2 * i] = h2_fma(lo, s[i], z[i]);
    out[2 * i + 1] = h2_fma(hi, s[i], z[i]);
  }
}
Q3T_DEV uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
Q3T_DEV uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
// How the key axis is divided: by `most` in all, as many CTAs to each of the
// call's `tiles` (of all kv heads) as the grid and the workspace have.
struct PromptSplit {
  int thr;    // sequences of more rows than this
  int most;   // 1: not divided
  float *parts;  // [CTA] m[256], l[256], o[D / 4][256][4]
};
template <typename F>
Q3T_DEV int split_count(const PromptSplit &sp, int num_seqs, int n_kv, F count) {
  if (sp.most <= 1) return 1;
  int tiles = 0;
  for (int q = threadIdx.x & 31; q < num_seqs; q += 32) tiles += count(q);
  tiles = max(__reduce_add_sync(0xffffffffu, tiles), 1);
  return max(1, min(32, sp.most / (tiles * n_kv)));
}

template <int D>
struct PromptCfg {
  static constexpr int G = D / 32, BLK = kv4_block_bytes(D), ROWS = 256, KEYS = 64, PAGES = KEYS / kKv4Page;
  static constexpr int THREADS = 20 * 32;
  static constexpr int PART = ROWS * (D + 2);  // floats
  static constexpr int QB = 128 * D * 2, KB = KEYS * D * 2, VB = D * KEYS * 2, PB = 128 * KEYS * 2;
  static constexpr int SC = PAGES * 2 * D;  // a tile's scales and zeros of K, or of V
  static constexpr int ST = 2, RING = 12 * D;  // blocks on their way to an unpacking warp: digits, scale entries
  static constexpr size_t kSmem =
      2 * QB + 2 * KB + 2 * VB + 4 * PB + 2 * SC + 2 * PAGES * ST * RING + 1024;  // from a 1024-byte boundary
};

template <int D>
__global__ void __launch_bounds__(PromptCfg<D>::THREADS, 1) k_kv4_prompt(const __grid_constant__ Kv4AttendArgs a, PromptSplit ks) {
  using Cfg = PromptCfg<D>;
  constexpr int G = Cfg::G, BLK = Cfg::BLK, ROWS = Cfg::ROWS, KEYS = Cfg::KEYS, PAGES = Cfg::PAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[25];
  uint64_t *k_full = bars, *v_full = bars + 2, *k_freed = bars + 4, *v_freed = bars + 6;  // by buffer
  uint64_t *s_full = bars + 8, *s_freed = bars + 12;                                     // by half and buffer
  // by half and buffer too, although O is one: a softmax thread may arrive for tile i + 1 before another has for tile i,
  // and a thread that asks for a phase may find one or two more done (a parity names only the next one)
  uint64_t *p_full = bars + 16, *pv_done = bars + 20, *q_full = bars + 24;
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float k_fac[8][PAGES], kk_fac[8][KEYS];  // 2^-power of a page of K, and of keys that have their own
  __shared__ __align__(16) float v_exp[2][PAGES], v_one[2][PAGES];     // of a page: V's power, and 2^-power
  __shared__ __align__(16) float vk_exp[2][KEYS], vk_one[2][KEYS];  // the same of every key
  __shared__ uint8_t k_bad[8][KEYS], v_bad[2][KEYS];  // a key's groups that are no numbers: any of K's; of V's, by bit
  // of a page: bit 0 it is there, bit 1 such groups, bit 2 its keys have powers of their own
  __shared__ __align__(4) uint8_t k_says[8][PAGES], v_says[2][PAGES];
  __shared__ int dead;  // a wait gave up
  uint8_t *base = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *sq = base, *sk = sq + 2 * Cfg::QB, *sv = sk + 2 * Cfg::KB, *sp = sv + 2 * Cfg::VB, *scales = sp + 4 * Cfg::PB,
          *rings = scales + 2 * Cfg::SC;
  pdl_wait();
  const int n_kv = a.c.n_kv, gq = a.n_heads / n_kv, kvh = blockIdx.x % n_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 17 && lane < 25) {
    // arrivals: the unpacking warps; both halves' products; the scores, and what K's warps say of the tile;
    // the softmax threads of a half; P V; all softmax threads
    const int n = lane < 4 ? PAGES : lane < 12 ? 2 : lane < 20 ? 128 : lane < 24 ? 1 : 256;
    mbar_init(&bars[lane], n);
    fence_mbar_init();
    if (lane == 0) dead = 0;
  }
  auto tiles_of = [&](int q) {
    int t0, n, pos0;
    seq_rows(a.b, q, t0, n, pos0);
    return n * gq > ks.thr ? (n * gq + ROWS - 1) / ROWS : 0;
  };
  const int splits = split_count(ks, a.b.num_seqs, n_kv, tiles_of), split = blockIdx.x / n_kv % splits;
  int s, i_rev;
  if (!find_item(a.b.num_seqs, blockIdx.x / n_kv / splits, tiles_of, s, i_rev)) return;
  int t0, n, pos0;
  seq_rows(a.b, s, t0, n, pos0);
  const int total = n * gq, row0 = ((total + ROWS - 1) / ROWS - 1 - i_rev) * ROWS;  // the longest tiles first
  const int nrow = min(ROWS, total - row0);
  const int pos_lo = pos0 + row0 / gq, pos_hi = pos0 + (row0 + nrow - 1) / gq;
  const int key_lo = first_key(pos_lo, a.window);
  int pg_lo = key_lo >> 4;
  // tiles of keys that the first 128 rows see, and the others; both begin at page pg_lo
  auto pages_to = [&](int pos) { return pos < 0 ? 0 : max(0, min((pos >> 4) + 1, a.c.table_stride) - pg_lo); };
  auto tiles_to = [&](int pos) { return (pages_to(pos) + PAGES - 1) / PAGES; };
  int nt0 = tiles_to(pos0 + (row0 + min(nrow, 128) - 1) / gq), nt1 = nrow > 128 ? tiles_to(pos_hi) : 0;
  int n_tiles = max(nt0, nt1), n_pages = pages_to(pos_hi);
  if (splits > 1) {  // this CTA's tiles of keys, four at least
    const int per = max(4, (n_tiles + splits - 1) / splits), skip = split * per;
    nt0 = max(0, min(nt0 - skip, per)), nt1 = max(0, min(nt1 - skip, per));
    n_tiles = max(nt0, nt1);
    pg_lo += skip * PAGES;
    n_pages = max(0, min(n_pages - skip * PAGES, per * PAGES));
    if (n_tiles == 0) {  // nothing left for it
      if ((int)threadIdx.x < nrow) {
        float *part = ks.parts + (size_t)blockIdx.x * Cfg::PART + threadIdx.x;
        part[0] = -INFINITY, part[ROWS] = 0.f;
      }
      return;
    }
  }

  if (warp == 16) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now may the next kernel start: one that took tensor memory and then
  // waited for this grid would keep a later CTA of it waiting for its own
  pdl_launch();
  const uint32_t tmem = tmem_slot;  // S of half h, buffer b: 128 h + 64 b; O of half h: 256 + 128 h
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    int n = 0;
#pragma unroll 1
    while (!mbar_try(bar, parity))
      if (++n > kMbarPolls || *(volatile int *)&dead) {
        *(volatile int *)&dead = 1;
        break;
      }
  };

  // row o of the tile is head hd of token tok of the sequence; o + rem0 is small, so 2^32 / gq, rounded up, divides it
  const int tok0 = row0 / gq, rem0 = row0 - tok0 * gq;
  const uint32_t inv_gq = gq == 1 ? 0u : 0xffffffffu / (uint32_t)gq + 1u;
  auto row_at = [&](int o, int &tok, int &hd) {
    const int x = rem0 + min(o, nrow - 1), y = gq == 1 ? x : (int)__umulhi((uint32_t)x, inv_gq);
    tok = tok0 + y;
    hd = kvh * gq + x - y * gq;
  };
  // Q's way in and O's way out: LPR lanes to a row, so that a warp's accesses are whole lines
  constexpr int LPR = D / 8, RPS = 32 / LPR;
  auto q_at = [&](int o, int c) {  // 16 bytes: dims 8 c .. of row o
    return reinterpret_cast<uint4 *>(sq + (o >> 7) * Cfg::QB + (c >> 3) * (128 * 128) + (o & 127) * 128 +
                                     (((c & 7) ^ (o & 7)) << 4));
  };
  float q_back = 0.f;  // softmax: what the scores' scale makes up for
  if (warp < 8) {
    // Q: f16 times a power of two per row, swizzled; a warp has the rows of its own threads
    const int c = lane % LPR, k0 = lane / LPR;
    int tok, hd;
    row_at(threadIdx.x, tok, hd);
    const long long mine = (long long)((size_t)(t0 + tok) * a.ldq + (size_t)hd * D);
    if (a.vec) {
#pragma unroll 8
      for (int k = 0; k < 32; k += RPS)
        cp_async16(q_at(32 * warp + k0 + k, c), a.q + __shfl_sync(0xffffffffu, mine, k0 + k) + 8 * c, 16);
    } else {
#pragma unroll 1
      for (int k = 0; k < 32; k += RPS) {
        const uint16_t *from = a.q + __shfl_sync(0xffffffffu, mine, k0 + k) + 8 * c;
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = from[2 * e] | (uint32_t)from[2 * e + 1] << 16;
        *q_at(32 * warp + k0 + k, c) = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    uint32_t most = 0u;  // of both halves of a word at once: without signs, bf16 are ordered as their bits
#pragma unroll 8
    for (int c8 = 0; c8 < D / 8; c8++) {
      const uint4 u = *q_at(threadIdx.x, c8);
      most = __vmaxu2(most, __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                     __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu)));
    }
    const float up = to_2p14(bf2f((uint16_t)max(most & 0xffffu, most >> 16)));
    const float f = a.scale == 0.f ? 0.f : a.scale < 0.f ? -up : up;
    q_back = a.scale == 0.f ? 1.f : fabsf(a.scale) * __uint_as_float((254u << 23) - __float_as_uint(up));  // / up
#pragma unroll 1
    for (int c8 = 0; c8 < D / 8; c8 += 4) {
      uint4 u[4];
#pragma unroll
      for (int k = 0; k < 4; k++) u[k] = *q_at(threadIdx.x, c8 + k);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t x[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = pack_f16x2(bf2f(x[e] & 0xffffu) * f, __uint_as_float(x[e] & 0xffff0000u) * f);
        *q_at(threadIdx.x, c8 + k) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    fence_proxy_async();
    mbar_arrive(q_full);
  }

  if (warp >= 8 && warp < 16) {
    // ---- unpack: page w of every tile ----
    constexpr int EPL = 16 * G / 32;  // scale entries of a lane
    const bool is_v = warp & 2;  // each scheduler has warps of one kind, and with them less code
    const int w = (warp & 1) + 2 * (warp >= 12), g = lane >> 2, t = lane & 3;
    uint8_t *sc = scales + (is_v ? Cfg::SC : 0) + w * 2 * D;
    uint8_t *ring = rings + (warp - 8) * Cfg::ST * Cfg::RING;
    uint64_t *freed = is_v ? v_freed : k_freed;
    int ids = -1;
    bool there = false;  // the page asked for last
    auto fetch = [&](int tile, uint8_t *to) {
      if (tile % 32 == 0) {  // this warp's page of the next 32 tiles, by lane
        const int p = (tile + lane) * PAGES + w;
        ids = p < n_pages ? page_of(a.c, a.b, s, pg_lo + p) : -1;
      }
      const int id = __shfl_sync(0xffffffffu, ids, tile % 32);
      there = id >= 0;
      if (id >= 0) {
        const uint8_t *blk = a.c.pool + ((size_t)id * n_kv + kvh) * BLK;
#pragma unroll
        for (int x = 0; x < 8 * D; x += 512) cp_async16(to + x + 16 * lane, blk + (is_v ? 8 * D : 0) + x + 16 * lane, 16);
        if (lane < D / 4) cp_async16(to + 8 * D + 16 * lane, blk + 16 * D + 16 * lane, 16);
      }
      cp_async_commit();
    };
    fetch(0, ring);
#pragma unroll 1
    for (int i = 0; i < n_tiles; i++) {
      const int b = i & 1, key0 = (pg_lo + i * PAGES + w) * 16;
      const bool here = there;
      const uint8_t *from = ring + b * Cfg::RING;
      cp_async_wait<0>();
      __syncwarp();  // all lanes' copies are here, and all lanes are done with the block before
      fetch(i + 1, ring + (b ^ 1) * Cfg::RING);
      // what no row sees, and what is no number, becomes zeros
      uint32_t en[EPL];
      float top = 0.f;
      uint32_t bad = 0;
#pragma unroll
      for (int x = 0; x < EPL; x++) {
        const int e = lane + 32 * x, c = 2 * (e >> 2 & 3) + (e & 1) + 8 * (e >> 1 & 1), key = key0 + c;  // group e / 16
        en[x] = *reinterpret_cast<const uint32_t *>(from + 8 * D + 8 * e + (is_v ? 4 : 0));
        if (!(here && key <= pos_hi && key >= key_lo)) en[x] = 0u;
        if ((en[x] & 0x7f80u) == 0x7f80u || (en[x] & 0x7f800000u) == 0x7f800000u) en[x] = 0u, bad |= 1u << (e >> 4);
        const float z = __uint_as_float(en[x] & 0xffff0000u);
        top = fmaxf(top, fmaxf(fabsf(z), fabsf(fmaf(15.f, bf2f(en[x] & 0xffffu), z))));
      }
      // (of values >= 0 the largest bits are the largest value's)
      top = fminf(top, FLT_MAX);
      const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
      bad |= __shfl_xor_sync(0xffffffffu, bad, 16);  // lanes l and l + 16 hold a token's groups
      const int some = __any_sync(0xffffffffu, bad != 0u), token = 16 * w + 2 * (lane >> 2 & 3) + (lane & 1) + 8 * (lane >> 1 & 1);
      // {s, z} in f16, where every lane finds them
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const int key = key0 + 2 * (lane >> 2 & 3) + (lane & 1) + 8 * (lane >> 1 & 1);
      const bool own_powers = __any_sync(0xffffffffu, here && key <= pos_hi && key >= key_lo && top < most * 0x1p-10f);
      if (!own_powers) top = most;
      float f = to_2p14(top);
      // A key of V that is zeros has a power that is small, so that it does not hold ref up, but lets l see its weight; no
      // power of V is so small that a sum of 2^15 2^-power leaves 32 bits.
      if (is_v) f = top == 0.f ? 0x1p60f : fminf(f, 0x1p90f);
#pragma unroll
      for (int x = 0; x < EPL; x++)
        *reinterpret_cast<uint32_t *>(sc + 4 * (lane + 32 * x)) =
            pack_f16x2(bf2f(en[x] & 0xffffu) * f, __uint_as_float(en[x] & 0xffff0000u) * f);
      __syncwarp();
      if (i >= 2) wait(&freed[b], ((i >> 1) - 1) & 1);
      if (is_v) {
        // rows are dims, one atom of 64 keys; digits of dims g and g + 8 of every 16.  A page's keys lie in the order
        // that a lane has them in (2t, 2t + 1, 2t + 8, 2t + 9; P's do too): half the stores
        uint8_t *to = sv + b * Cfg::VB + g * 128 + (((2 * w + (t >> 1)) ^ g) << 4) + 8 * (t & 1);
#pragma unroll 1
        for (int j = 0; j < G; j++, to += 32 * 128) {
          const uint4 u = *reinterpret_cast<const uint4 *>(sc + 64 * j + 16 * t);  // keys 2t, 2t + 1, 2t + 8, 2t + 9
          const uint2 d = *reinterpret_cast<const uint2 *>(from + 512 * (j >> 1) + 16 * lane + 8 * (j & 1));
          const uint32_t sx[2] = {lows(u.x, u.y), lows(u.z, u.w)}, zx[2] = {highs(u.x, u.y), highs(u.z, u.w)};
#pragma unroll
          for (int m = 0; m < 2; m++) {
            uint32_t o[4];
            unpack8(m ? d.y : d.x, sx, zx, o);  // (dim g, dim g + 8) x (keys 2t .., keys 2t + 8 ..)
            *reinterpret_cast<uint2 *>(to + 16 * m * 128) = make_uint2(o[0], o[2]);
            *reinterpret_cast<uint2 *>(to + (16 * m + 8) * 128) = make_uint2(o[1], o[3]);
          }
        }
        if (lane < 16) {
          v_bad[b][token] = (uint8_t)bad;
          vk_exp[b][token] = (float)-exponent(f), vk_one[b][token] = f;
        }
        if (lane == 0) {
          v_says[b][w] = (uint8_t)(2 * some + 4 * own_powers);
          v_exp[b][w] = (float)-exponent(f), v_one[b][w] = f;
        }
      } else {
        // rows are keys, D / 64 atoms of 64 dims; digits of keys g and g + 8
        uint8_t *to = sk + b * Cfg::KB + (16 * w + g) * 128;
#pragma unroll 1
        for (int j = 0; j < G; j++) {
          const int c = 4 * j + t, at = (c >> 3) * (KEYS * 128) + (((c & 7) ^ g) << 4);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t sz = *reinterpret_cast<const uint32_t *>(sc + 64 * j + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
            const uint32_t d = *reinterpret_cast<const uint32_t *>(from + 4 * D * h + 4 * G * lane + 4 * j);
            const uint32_t s1 = lows(sz, sz), z1 = highs(sz, sz), sx[2] = {s1, s1}, zx[2] = {z1, z1};
            uint32_t o[4];
            unpack8(d, sx, zx, o);
            *reinterpret_cast<uint4 *>(to + 8 * 128 * h + at) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        // Eight deep: a softmax reads these of tile i after its scores have freed K.
        // K of tile i + 7 waits for a score of tile i + 5, that for a softmax to be
        // done with tile i + 2, that for V, which waits for every P V of tile i.
        if (lane < 16) k_bad[i & 7][token] = bad != 0u;
        if (own_powers && lane < 16) kk_fac[i & 7][token] = 1.f / f;
        if (lane == 0) {
          k_fac[i & 7][w] = 1.f / f;
          k_says[i & 7][w] = (uint8_t)(here + 2 * some + 4 * own_powers);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(is_v ? &v_full[b] : &k_full[b]);
    }
    cp_async_wait<0>();
  } else if (warp >= 16) {
    // ---- products: a warp to each half's S and to its P V, one lane of it ----
    const int h = warp & 1, nt = h ? nt1 : nt0, other = h ? nt0 : nt1;
    if (lane == 0 && warp < 18) {
      constexpr uint32_t id_s = umma_idesc_f16(128, KEYS);
      const uint64_t dq = sw128_desc(sq + h * Cfg::QB), dk = sw128_desc(sk);
      if (nt > 0) wait(q_full, 0);
      for (int i = 0; i < nt; i++) {
        const int b = i & 1;
        wait(&k_full[b], (i >> 1) & 1);
        if (i >= 2) wait(&s_freed[2 * h + b], ((i >> 1) - 1) & 1);
        if (*(volatile int *)&dead) break;
        mbar_arrive(&s_full[2 * h + b]);
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; k++)
          umma_kf16(tmem + 128 * h + KEYS * b, dq + (((k >> 2) * (128 * 128) + 32 * (k & 3)) >> 4),
                    dk + ((b * Cfg::KB + (k >> 2) * (KEYS * 128) + 32 * (k & 3)) >> 4), id_s, k > 0);
        umma_commit(&s_full[2 * h + b]);
        umma_commit(&k_freed[b]);
        if (i >= other) umma_commit(&k_freed[b]);  // the other half has no use for this tile
      }
    } else if (lane == 0) {
      constexpr uint32_t id_o = umma_idesc_f16(128, D);
      const uint64_t dp = sw128_desc(sp + 2 * h * Cfg::PB), dv = sw128_desc(sv);
      for (int i = 0; i < nt; i++) {
        const int b = i & 1;
        wait(&v_full[b], (i >> 1) & 1);
        wait(&p_full[2 * h + b], (i >> 1) & 1);
        if (*(volatile int *)&dead) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < KEYS / 16; k++)
          umma_kf16(tmem + 256 + 128 * h, dp + ((b * Cfg::PB + 32 * k) >> 4), dv + ((b * Cfg::VB + 32 * k) >> 4), id_o,
                    i > 0 || k > 0);
        umma_commit(&pv_done[2 * h + b]);
        umma_commit(&v_freed[b]);
        if (i >= other) umma_commit(&v_freed[b]);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: a thread holds row r of half h ----
    const int h = threadIdx.x >> 7, r = threadIdx.x & 127, nt = h ? nt1 : nt0;
    int tok, hd;
    row_at(threadIdx.x, tok, hd);
    const int lim = pos0 + tok, low = first_key(lim, a.window);
    // keys that all rows of this half see
    const int all_to = pos0 + (row0 + min(128 * h, nrow - 1)) / gq;
    const int all_from = first_key(pos0 + (row0 + min(128 * h + 127, nrow - 1)) / gq, a.window);
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, t_s = tmem + lanes + 128 * h, t_o = tmem + lanes + 256 + 128 * h;
    uint8_t *my_p = sp + 2 * h * Cfg::PB + r * 128;
    float ref = -INFINITY, l = 0.f;  // ref: what exponents are taken from, those of O and l
    uint32_t nan = 0;              // of the keys this row has seen: bit j, V of group j; bit 7, K
#pragma unroll 1
    for (int i = 0; i < nt; i++) {
      const int b = i & 1, q = i & 7, key0 = (pg_lo + i * PAGES) * 16;
      wait(&s_full[2 * h + b], (i >> 1) & 1);
      tc_fence_after();
      uint32_t x[2][32];
      tmem_ld32_async(t_s + KEYS * b, x[0]);
      tmem_ld32_async(t_s + KEYS * b + 32, x[1]);
      const uint32_t k_say = *reinterpret_cast<const uint32_t *>(k_says[q]);
      const float4 k4 = *reinterpret_cast<const float4 *>(k_fac[q]);
      const bool edge = key0 + KEYS - 1 > all_to || key0 < all_from || (k_say & 0x05050505u) != 0x01010101u;
      // a score of page p is its column times f[p]; zero rows and pages keep it off 0 and infinity
      float f[PAGES] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int p = 0; p < PAGES; p++) f[p] = fminf(fmaxf(q_back * f[p], 0x1p-100f), 0x1p100f);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&s_freed[2 * h + b]);
      uint32_t see[2] = {0xffffffffu, 0xffffffffu};
      if (edge) {
        if (k_say & 0x04040404u) {  // keys' own powers into their scores
#pragma unroll
          for (int k = 0; k < KEYS; k++) {
            const float own = fminf(fmaxf(q_back * kk_fac[q][k], 0x1p-100f), 0x1p100f);
            x[k >> 5][k & 31] =
                __float_as_uint(__uint_as_float(x[k >> 5][k & 31]) * (k_say >> (8 * (k >> 4) + 2) & 1 ? own : f[k >> 4]));
          }
#pragma unroll
          for (int p = 0; p < PAGES; p++) f[p] = 1.f;
        }
        // bits of the keys that this row sees
        const int last = lim - key0, first = low - key0;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int l1 = last - 32 * c, f1 = first - 32 * c;
          uint32_t y = l1 < 0 ? 0u : 0xffffffffu >> (31 - min(l1, 31));
          y = f1 > 31 ? 0u : y & 0xffffffffu << max(f1, 0);
          if (!(k_say >> 16 * c & 1)) y &= 0xffff0000u;
          if (!(k_say >> (16 * c + 8) & 1)) y &= 0xffffu;
          see[c] = y;
#pragma unroll
          for (int k = 0; k < 32; k++)
            if (!(y >> k & 1)) x[c][k] = 0xff800000u;
        }
      }
      float most[PAGES];  // of a page's scores
      auto largest = [&] {
#pragma unroll
        for (int p = 0; p < PAGES; p++) {
          float y = __uint_as_float(x[p >> 1][16 * (p & 1)]);
#pragma unroll
          for (int k = 1; k < 16; k++) y = fmaxf(y, __uint_as_float(x[p >> 1][16 * (p & 1) + k]));
          most[p] = y * f[p];
        }
      };
      largest();
      wait(&v_full[b], (i >> 1) & 1);  // which means too that P V of tile i - 2 has been, and P may be written
      const uint32_t v_say = *reinterpret_cast<const uint32_t *>(v_says[b]);
      const float4 v4 = *reinterpret_cast<const float4 *>(v_exp[b]), o4 = *reinterpret_cast<const float4 *>(v_one[b]);
      float ve[PAGES] = {v4.x, v4.y, v4.z, v4.w}, one[PAGES] = {o4.x, o4.y, o4.z, o4.w};
      const bool own_powers = v_say & 0x04040404u;
      if (own_powers) {  // V's powers into the scores, key by key
#pragma unroll
        for (int k = 0; k < KEYS; k += 4) {
          const float4 e = *reinterpret_cast<const float4 *>(&vk_exp[b][k]);
          uint32_t *y = &x[k >> 5][k & 31];
          const uint64_t ff = f2_pack(f[k >> 4], f[k >> 4]);
          float y0, y1, y2, y3;
          f2_split(f2_fma(f2_pack(__uint_as_float(y[0]), __uint_as_float(y[1])), ff, f2_pack(e.x, e.y)), y0, y1);
          f2_split(f2_fma(f2_pack(__uint_as_float(y[2]), __uint_as_float(y[3])), ff, f2_pack(e.z, e.w)), y2, y3);
          y[0] = __float_as_uint(y0), y[1] = __float_as_uint(y1), y[2] = __float_as_uint(y2), y[3] = __float_as_uint(y3);
        }
#pragma unroll
        for (int p = 0; p < PAGES; p++) f[p] = 1.f, ve[p] = one[p] = 0.f;  // (l has its share below)
        largest();
      }
      if ((k_say | v_say) & 0x02020202u)
#pragma unroll 1
        for (int k = 0; k < KEYS; k++)
          if (see[k >> 5] >> (k & 31) & 1) nan |= v_bad[b][k] | (uint32_t)k_bad[q][k] << 7;
      float scale_o = 1.f, top = -INFINITY;
      bool move = false;
#pragma unroll
      for (int p = 0; p < PAGES; p++) top = fmaxf(top, most[p] + ve[p]);
      if (top > ref + 15.f) {  // the first time, or past what P is to hold
        const float to = top - 7.f;
        scale_o = ref == -INFINITY ? 0.f : ex2(ref - to);
        ref = to;
        l *= scale_o;
        move = true;
      }
      const float mu = ref == -INFINITY ? 0.f : ref;
#pragma unroll
      for (int p = 0; p < PAGES; p++) {
        const float c0 = ve[p] - mu;
        const uint64_t ff = f2_pack(f[p], f[p]), cc = f2_pack(c0, c0);
        uint64_t part = 0;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int at = 16 * (p & 1) + 4 * c + 8 * (k & 1) + 2 * (k >> 1);  // V's order of keys
            float y0, y1;
            f2_split(f2_fma(f2_pack(__uint_as_float(x[p >> 1][at]), __uint_as_float(x[p >> 1][at + 1])), ff, cc), y0, y1);
            y0 = ex2(y0), y1 = ex2(y1);
            part = f2_add(part, f2_pack(y0, y1));
            w[k] = pack_f16x2(y0, y1);
            x[p >> 1][at] = __float_as_uint(y0), x[p >> 1][at + 1] = __float_as_uint(y1);
          }
          *reinterpret_cast<uint4 *>(my_p + b * Cfg::PB + (((2 * p + c) ^ (r & 7)) << 4)) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
        float s0, s1;
        f2_split(part, s0, s1);
        l = fmaf(s0 + s1, one[p], l);
      }
      if (own_powers) {
        uint64_t sum = 0;
#pragma unroll
        for (int k = 0; k < KEYS; k += 4) {
          const float4 o = *reinterpret_cast<const float4 *>(&vk_one[b][k]);
          const uint32_t *y = &x[k >> 5][k & 31];
          sum = f2_fma(f2_pack(__uint_as_float(y[0]), __uint_as_float(y[1])), f2_pack(o.x, o.y), sum);
          sum = f2_fma(f2_pack(__uint_as_float(y[2]), __uint_as_float(y[3])), f2_pack(o.z, o.w), sum);
        }
        float s0, s1;
        f2_split(sum, s0, s1);
        l += s0 + s1;
      }
      if (i > 0 && __any_sync(0xffffffffu, move)) {
        wait(&pv_done[2 * h + (b ^ 1)], ((i - 1) >> 1) & 1);  // O is whole
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; c++) {
          tmem_ld32_async(t_o + 32 * c, x[0]);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k++) x[0][k] = __float_as_uint(__uint_as_float(x[0][k]) * scale_o);
          tmem_st32(t_o + 32 * c, x[0]);
        }
      }
      tc_fence_before();
      fence_proxy_async();
      mbar_arrive(&p_full[2 * h + b]);
    }
    if (nt > 0) wait(&pv_done[2 * h + ((nt - 1) & 1)], ((nt - 1) >> 1) & 1);
    tc_fence_after();
    const bool gone = *(volatile int *)&dead;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float *part = splits > 1 ? ks.parts + (size_t)blockIdx.x * Cfg::PART + threadIdx.x : nullptr;
    const bool in_tile = (int)threadIdx.x < nrow;
    // a part weighs l 2^ref, here as a number of kPartL and an exponent: ref has V's powers, which may be far apart
    if (part && in_tile) {
      const int e = l == 0.f ? 0 : min(max(exponent(l) - kPartL, -126), 126);
      part[0] = ref + (float)e;
      part[ROWS] = gone ? __uint_as_float(0x7fc00000u) : l * __uint_as_float((uint32_t)(127 - e) << 23);
    }
#pragma unroll 1
    for (int c = 0; c < D / 32; c++) {
      uint32_t x[32];
      if (nt > 0) {
        tmem_ld32_async(t_o + 32 * c, x);
        tmem_wait_ld();
      }
      else {
#pragma unroll
        for (int k = 0; k < 32; k++) x[k] = 0u;
      }
      const bool is_nan = gone || (nan >> 7 & 1) || (nan >> c & 1);
      const float f1 = is_nan ? __uint_as_float(0x7fc00000u) : inv;
      if (part) {
        float4 *to = reinterpret_cast<float4 *>(part - threadIdx.x + 2 * ROWS) + threadIdx.x;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (in_tile) to[(8 * c + k) * ROWS] = make_float4(__uint_as_float(x[4 * k]) * f1, __uint_as_float(x[4 * k + 1]) * f1,
                                               __uint_as_float(x[4 * k + 2]) * f1, __uint_as_float(x[4 * k + 3]) * f1);
        continue;
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
          y[e] = pack_bf16x2(__uint_as_float(x[8 * k + 2 * e]) * f1, __uint_as_float(x[8 * k + 2 * e + 1]) * f1);
        *q_at(threadIdx.x, 4 * c + k) = make_uint4(y[0], y[1], y[2], y[3]);  // (this half's S are done with Q)
      }
    }
    __syncwarp();
    const int c = lane % LPR, k0 = lane / LPR;
    const long long mine = (long long)((size_t)(t0 + tok) * a.ldo + (size_t)hd * D);
    if (part) {
      // k_kv4_join has the rest
    } else if (a.vec) {
#pragma unroll 8
      for (int k = 0; k < 32; k += RPS) {
        const uint4 u = *q_at(32 * warp + k0 + k, c);
        uint16_t *to = a.out + __shfl_sync(0xffffffffu, mine, k0 + k) + 8 * c;
        if (32 * warp + k0 + k < nrow) *reinterpret_cast<uint4 *>(to) = u;
      }
    } else {
#pragma unroll 1
      for (int k = 0; k < 32; k += RPS) {
        const uint4 u = *q_at(32 * warp + k0 + k, c);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
        uint16_t *to = a.out + __shfl_sync(0xffffffffu, mine, k0 + k) + 8 * c;
        if (32 * warp + k0 + k < nrow)
#pragma unroll
          for (int e = 0; e < 8; e++) to[e] = (uint16_t)(x[e >> 1] >> 16 * (e & 1));
      }
    }
    if (gone && threadIdx.x == 0 && a.err) atomicOr(a.err, 0x400);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    if (dead) __nanosleep(50000);  // products that were issued before a wait gave up end within it
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of k_kv4_prompt's tiles, where it divided the keys: a thread
// has a row, eight dims of it (32 to a thread, one part after the other, took
// 33 us for 18 parts: all of it waiting for loads).  A part's o is divided by
// its l already, so a part weighs l 2^m (l as kPartL has it); parts come in
// order, and the result does not depend on timing.
template <int D>
__global__ void __launch_bounds__(256) k_kv4_join(const __grid_constant__ Kv4AttendArgs a, PromptSplit sp) {
  using Cfg = PromptCfg<D>;
  constexpr int ROWS = Cfg::ROWS;
  pdl_wait();
  pdl_launch();
  const int n_kv = a.c.n_kv, gq = a.n_heads / n_kv, kvh = blockIdx.x % n_kv;
  auto tiles_of = [&](int q) {
    int t0, n, pos0;
    seq_rows(a.b, q, t0, n, pos0);
    return n * gq > sp.thr ? (n * gq + ROWS - 1) / ROWS : 0;
  };
  const int splits = split_count(sp, a.b.num_seqs, n_kv, tiles_of);
  if (splits == 1) return;
  int s, i_rev;
  if (!find_item(a.b.num_seqs, blockIdx.x / n_kv, tiles_of, s, i_rev)) return;
  int t0, n, pos0;
  seq_rows(a.b, s, t0, n, pos0);
  const int total = n * gq, row0 = ((total + ROWS - 1) / ROWS - 1 - i_rev) * ROWS, nrow = min(ROWS, total - row0);
  for (int at = blockIdx.y * 256 + threadIdx.x; at < nrow * (D / 8); at += gridDim.y * 256) {
    const int d0 = 8 * (at / nrow), r = at % nrow, flat = row0 + r, tok = flat / gq;
    const float *part = sp.parts + (size_t)(blockIdx.x / n_kv * splits * n_kv + kvh) * Cfg::PART + r;
    const size_t step = (size_t)n_kv * Cfg::PART;
    constexpr int N = 8;  // parts whose loads are on their way together
    float M = -INFINITY, L = 0.f;
    for (int k0 = 0; k0 < splits; k0 += N) {
      float m[N];
#pragma unroll
      for (int k = 0; k < N; k++) m[k] = k0 + k < splits ? part[(k0 + k) * step] : -INFINITY;
#pragma unroll
      for (int k = 0; k < N; k++) M = fmaxf(M, m[k]);
    }
    float o[8] = {};
    for (int k0 = 0; k0 < splits; k0 += N) {
      float m[N], l[N];
      float4 u[N], v[N];
#pragma unroll
      for (int k = 0; k < N; k++) {
        const float *p = part + (k0 + k) * step;
        m[k] = k0 + k < splits ? p[0] : 0.f, l[k] = k0 + k < splits ? p[ROWS] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < N; k++) {
        const float4 *from = reinterpret_cast<const float4 *>(part - r + (k0 + k) * step + 2 * ROWS) + r + (size_t)(d0 / 4) * ROWS;
        u[k] = v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (l[k] != 0.f) u[k] = from[0], v[k] = from[ROWS];  // it has keys of this row
      }
#pragma unroll
      for (int k = 0; k < N; k++) {
        const float w = l[k] == 0.f ? 0.f : l[k] * ex2(m[k] - M);
        L += w;
        o[0] = fmaf(w, u[k].x, o[0]), o[1] = fmaf(w, u[k].y, o[1]), o[2] = fmaf(w, u[k].z, o[2]), o[3] = fmaf(w, u[k].w, o[3]);
        o[4] = fmaf(w, v[k].x, o[4]), o[5] = fmaf(w, v[k].y, o[5]), o[6] = fmaf(w, v[k].z, o[6]), o[7] = fmaf(w, v[k].w, o[7]);
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] *= inv;
    store8(a.out + (size_t)(t0 + tok) * a.ldo + (size_t)(kvh * gq + flat - tok * gq) * D + d0, a.vec, o);
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*k)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, bool pdl, cudaStream_t st,
                   Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  if (pdl && g_use_pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...);
  if (e == cudaSuccess) g_launches++;
  return e;
}

// Once per device: shared-memory limits and clusters of 16.
template <typename F>
cudaError_t once_per_device(std::atomic<uint64_t> &done, F &&f) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  if ((e = f()) != cudaSuccess) return e;
  done.fetch_or(bit, std::memory_order_release);
  return cudaSuccess;
}

// Head splits that give a launch a few CTAs per SM where there are few windows.
int head_splits(int windows, int n_kv) {
  int s = 1;
  while (s < n_kv && (int64_t)windows * s < 444) s *= 2;
  return s < n_kv ? s : n_kv;
}

template <typename T, int D, int E>
cudaError_t append_launch(const Kv4AppendArgs &a, int windows, cudaStream_t st, bool pdl) {
  static std::atomic<uint64_t> done{0};
  const int per = (a.c.n_kv + a.splits - 1) / a.splits;
  const size_t smem = (size_t)per * kv4_block_bytes(D);
  cudaError_t e = once_per_device(done, [] {
    return cudaFuncSetAttribute(k_kv4_append<T, D, E>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10);
  });
  if (e != cudaSuccess) return e;
  return launch(k_kv4_append<T, D, E>, dim3(windows, a.splits), kAppendThreads, smem, 1, pdl, st, a);
}

template <int D>
cudaError_t read_launch(const Kv4ReadArgs &a, int windows, cudaStream_t st, bool pdl) {
  static std::atomic<uint64_t> done{0};
  const int per = (a.c.n_kv + a.splits - 1) / a.splits;
  cudaError_t e = once_per_device(done, [] {
    return cudaFuncSetAttribute(k_kv4_read<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10);
  });
  if (e != cudaSuccess) return e;
  return launch(k_kv4_read<D>, dim3(windows, a.splits), kReadThreads, (size_t)per * kv4_block_bytes(D), 1, pdl, st, a);
}

template <int D, int NT>
cudaError_t attend_launch(const Kv4AttendArgs &a0, int rows, int max_kv, void *ws, int64_t ws_bytes, cudaStream_t st, bool pdl) {
  using Cfg = AttendCfg<D, NT>;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> resident{0};  // CTAs that one device holds at once
  cudaError_t e = once_per_device(done, [] {
    cudaError_t r = cudaFuncSetAttribute(k_kv4_attend<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg::smem(Cfg::MAXSEQ));
    int dev = 0, sms = 0, occ = 0;
    if (r == cudaSuccess) r = cudaGetDevice(&dev);
    if (r == cudaSuccess) r = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (r == cudaSuccess)
      r = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, k_kv4_attend<D, NT>, Cfg::W * 32, Cfg::smem(256));
    if (r == cudaSuccess) resident.store(sms * std::max(occ, 1));
    return r;
  });
  if (e != cudaSuccess) return e;
  Kv4AttendArgs a = a0;
  a.units = std::max(1, (rows + Cfg::R - 1) / Cfg::R);
  constexpr int kUnits = Cfg::MAXSEQ;
  if (a0.b.num_seqs * (int64_t)a.units > kUnits) {  // a part of the sequences at a time
    const int at_once = kUnits / a.units;
    for (int s0 = 0; s0 < a0.b.num_seqs; s0 += at_once) {
      a.b.num_seqs = std::min(at_once, a0.b.num_seqs - s0);
      a.b.q_start = a0.b.q_start + s0;
      a.b.kv_len = a0.b.kv_len + s0;
      if (a0.b.table_row) a.b.table_row = a0.b.table_row + s0;
      a.b.first = a0.b.first + s0;
      if ((e = attend_launch<D, NT>(a, rows, max_kv, ws, ws_bytes, st, pdl)) != cudaSuccess) return e;
    }
    return cudaSuccess;
  }
  // one grid that fills the GPU once, fewer where a warp would have less than one step
  const bool windowed = a.window > 0 && (max_kv <= 0 || a.window < max_kv);
  const int64_t keys = windowed ? (int64_t)a.window + 31 : max_kv > 0 ? max_kv : 1 << 20;
  const int64_t pages = std::min<int64_t>(keys / 16 + 1, a.c.table_stride);
  const int64_t units = (int64_t)a.b.num_seqs * a.units, steps = (pages + 1) / 2 * units;
  // A CTA to each unit of each kv head where they all fit the GPU at once and a warp's share is short: no second
  // launch to join parts.  The more CTAs, the less an equal division gains (us, whole against divided, D = 128): 8 CTAs
  // of 200 keys 6.8 and 8.2, of 1000 12.1 and 8.7; 32 of 500 9.2 and 9.0; 128 of 500 9.4 and 12.3, of 1000 12.7 and
  // 15.3, of 2500 23.7 and 20.4; 512, which do not fit, of 500 21.5 and 20.1.
  const int64_t per_warp = ((pages + 1) / 2 + Cfg::W - 1) / Cfg::W, whole = units * a.c.n_kv;
  if (whole <= resident.load() && per_warp <= 2 + whole / 9)
    return launch(k_kv4_attend<D, NT>, dim3((unsigned)whole), Cfg::W * 32, Cfg::smem(1), 1, pdl, st, a, (PartNote *)nullptr,
                  (float *)nullptr);
  const int64_t fit = ws_bytes / (int64_t)(sizeof(PartNote) + 2 * Cfg::PART * 4);
  const int64_t most = std::min<int64_t>(std::min<int64_t>(resident.load(), fit) / a.c.n_kv, (steps + Cfg::W - 1) / Cfg::W);
  const int ctas = (int)std::max<int64_t>(most, 1), grid = ctas * a.c.n_kv;  // of a kv head, of all
  PartNote *notes = (PartNote *)ws;
  float *parts = (float *)(notes + grid);
  e = launch(k_kv4_attend<D, NT>, dim3(grid), Cfg::W * 32, Cfg::smem((int)units), 1, pdl, st, a, notes, parts);
  if (e != cudaSuccess || ctas == 1) return e;
  return launch(k_kv4_combine<D, NT>, dim3(grid), 256, 0, 1, false, st, a, (const PartNote *)notes, (const float *)parts);
}

}  // namespace

cudaError_t kv4_append(const Kv4AppendArgs &a0, bool f32_rows, cudaStream_t st, bool pdl) {
  const int windows = max_windows(a0.b);
  if (windows <= 0 || a0.b.num_seqs <= 0) return cudaSuccess;
  Kv4AppendArgs a = a0;
  a.splits = head_splits(windows, a.c.n_kv);
  // a split's blocks have to fit shared memory
  while ((size_t)((a.c.n_kv + a.splits - 1) / a.splits) * kv4_block_bytes(a.c.head_dim) > (40 << 10)) a.splits++;
  // a whole group to a lane where prompts fill their pages
  const bool deep = a.b.num_tokens >= kAppendDeep * a.b.num_seqs &&
                    (a.rope.rot == 0 || a.rope.interleaved || a.rope.rot == a.c.head_dim);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return deep ? append_launch<T, D, D / 32>(a, windows, st, pdl) : append_launch<T, D, 1>(a, windows, st, pdl);
  };
  if (a.c.head_dim == 128)
    return f32_rows ? go(0.f, std::integral_constant<int, 128>{}) : go((uint16_t)0, std::integral_constant<int, 128>{});
  return f32_rows ? go(0.f, std::integral_constant<int, 64>{}) : go((uint16_t)0, std::integral_constant<int, 64>{});
}

cudaError_t kv4_read(const Kv4ReadArgs &a0, cudaStream_t st, bool pdl) {
  const int windows = max_windows(a0.b);
  if (windows <= 0 || a0.b.num_seqs <= 0) return cudaSuccess;
  Kv4ReadArgs a = a0;
  a.splits = head_splits(windows, a.c.n_kv);
  while ((size_t)((a.c.n_kv + a.splits - 1) / a.splits) * kv4_block_bytes(a.c.head_dim) > (40 << 10)) a.splits++;
  return a.c.head_dim == 128 ? read_launch<128>(a, windows, st, pdl) : read_launch<64>(a, windows, st, pdl);
}

template <int D>
static cudaError_t prompt_launch(const Kv4AttendArgs &a, int thr, void *ws, int64_t ws_bytes, cudaStream_t st, bool pdl) {
  using Cfg = PromptCfg<D>;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> sms{0};
  cudaError_t e = once_per_device(done, [] {
    int dev = 0, n = 0;
    cudaError_t r = cudaFuncSetAttribute(k_kv4_prompt<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmem);
    if (r == cudaSuccess) r = cudaGetDevice(&dev);
    if (r == cudaSuccess) r = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (r == cudaSuccess) sms.store(n);
    return r;
  });
  if (e != cudaSuccess) return e;
  // tiles, at most: whole ones, and one more for every sequence that has over thr rows
  const int64_t rows = (int64_t)a.b.num_tokens * (a.n_heads / a.c.n_kv);
  const int64_t tiles = std::min<int64_t>(rows / Cfg::ROWS + std::min<int64_t>(a.b.num_seqs, rows / (thr + 1)), rows);
  if (tiles == 0) return cudaSuccess;  // too few rows for a sequence of over thr
  // where these cannot fill the GPU, CTAs share the keys of each
  const int64_t fit = std::min<int64_t>(sms.load(), ws_bytes / (4 * Cfg::PART));
  const int64_t grid = std::max<int64_t>(tiles * a.c.n_kv, fit);
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const PromptSplit sp = {thr, tiles * a.c.n_kv < fit ? (int)fit : 1, (float *)ws};
  e = launch(k_kv4_prompt<D>, dim3((unsigned)grid), Cfg::THREADS, Cfg::kSmem, 1, pdl, st, a, sp);
  if (e != cudaSuccess || sp.most == 1) return e;
  // as many CTAs as the GPU holds at once: more of them cost a call with nothing to join 9 us instead of 4
  const int64_t most = std::min(tiles * a.c.n_kv, fit / 2);
  const unsigned along = (unsigned)std::max<int64_t>(1, std::min<int64_t>(D / 8, 2 * sms.load() / most));
  return launch(k_kv4_join<D>, dim3((unsigned)most, along), 256, 0, 1, false, st, a, sp);
}

cudaError_t kv4_attend(const Kv4AttendArgs &a0, int max_q, int max_kv, void *ws, int64_t ws_bytes, cudaStream_t st,
                       bool pdl) {
  if (a0.b.num_tokens <= 0 || a0.b.num_seqs <= 0) return cudaSuccess;
  Kv4AttendArgs a = a0;
  const int gq = a.n_heads / a.c.n_kv;
  // Sequences of more rows than this go by tiles on k_kv4_prompt.  With 32 rows it takes, against k_kv4_attend (us,
  // group of 2, D = 128), 30 and 33 (one sequence of 8000 keys), 107 and 162 (eight), 132 and 189 (64 of 1000), but 22 and
  // 16 with one of 1000; with 16 rows k_kv4_attend takes 23, 88 and 104, and a tile as long as with 32.
  constexpr int kBig = 16;
  const bool some_big = max_q <= 0 || (int64_t)max_q * gq > kBig;
  // No sequence is small where all but one at their most leave more than kBig rows for the last.  Elsewhere both
  // kernels run, each for its sequences: a tile of 256 rows for one row of a decoding request costs 7 us of an SM.
  const bool none_small = (int64_t)a.b.num_tokens - (int64_t)(a.b.num_seqs - 1) * std::max(max_q, 0) > kBig / gq &&
                          (max_q > 0 || a.b.num_seqs == 1);
  if (some_big) {
    const int thr = none_small ? 0 : kBig;
    const cudaError_t e = a.c.head_dim == 128 ? prompt_launch<128>(a, thr, ws, ws_bytes, st, pdl)
                                              : prompt_launch<64>(a, thr, ws, ws_bytes, st, pdl);
    if (e != cudaSuccess || none_small || gq > kBig) return e;  // (one row of a group of over kBig is no small sequence)
    a.big = kBig;
  }
  const int rows = (some_big ? 1 : max_q) * gq;  // rows of a kv head: one column tile, or two
  if (a.c.head_dim == 128)
    return rows <= 2 ? attend_launch<128, 1>(a, rows, max_kv, ws, ws_bytes, st, pdl)
                     : attend_launch<128, 2>(a, rows, max_kv, ws, ws_bytes, st, pdl);
  return rows <= 4 ? attend_launch<64, 1>(a, rows, max_kv, ws, ws_bytes, st, pdl)
                   : attend_launch<64, 2>(a, rows, max_kv, ws, ws_bytes, st, pdl);
}

}  // namespace q3t

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
namespace {

using namespace q3t;

// the calling thread's current device is put back on every return
struct DeviceScope {
  int dev = -1;
  explicit DeviceScope(int want) {
    CK(cudaGetDevice(&dev));
    if (dev == want)
      dev = -1;
    else
      CK(cudaSetDevice(want));
  }
  ~DeviceScope() {
    if (dev >= 0) cudaSetDevice(dev);
  }
};

template <class F>
q3t_status guarded(F &&f) {
  try {
    f();
    return Q3T_OK;
  } catch (const Status &s) {
    return s.code;
  } catch (const CudaFail &c) {
    set_error("CUDA error %s (%s) in %s", cudaGetErrorName(c.err), cudaGetErrorString(c.err), c.what.c_str());
    return Q3T_CUDA_ERROR;
  } catch (const std::exception &e) {
    set_error("%s", e.what());
    return Q3T_CUDA_ERROR;
  }
}

bool aligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

Kv4View view_of(const char *what, const q3t_kv4_cache *c) {
  if (!c) FAIL(Q3T_INVALID_INPUT, "%s: null cache", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    FAIL(Q3T_INVALID_INPUT, "%s: head_dim %d (64 and 128 are built)", what, c->head_dim);
  if (c->num_kv_heads < 1 || c->num_kv_heads > 1024)
    FAIL(Q3T_INVALID_INPUT, "%s: num_kv_heads %d outside 1..1024", what, c->num_kv_heads);
  if (c->num_pages < 1 || c->num_pages > 0x7fffffff)
    FAIL(Q3T_INVALID_INPUT, "%s: num_pages %lld outside 1..2^31-1", what, (long long)c->num_pages);
  if (c->table_rows < 1 || c->table_stride < 1 || c->table_stride > (1 << 20))
    FAIL(Q3T_INVALID_INPUT, "%s: page table of %d x %d (1..2^20 entries to a row)", what, c->table_rows,
         c->table_stride);
  if (!c->pool || !c->page_table) FAIL(Q3T_INVALID_INPUT, "%s: null pool or page table", what);
  if (!aligned(c->pool, 16)) FAIL(Q3T_INVALID_INPUT, "%s: the pool must start on a 16-byte boundary", what);
  if (!aligned(c->page_table, 4)) FAIL(Q3T_INVALID_INPUT, "%s: the page table is not aligned to its entries", what);
  return Kv4View{(uint8_t *)c->pool, c->page_table, c->num_pages, c->num_kv_heads, c->head_dim, c->table_rows,
                 c->table_stride};
}

Kv4Batch batch_of(const char *what, const q3t_kv4_batch *b) {
  if (!b) FAIL(Q3T_INVALID_INPUT, "%s: null batch", what);
  if (b->num_seqs < 0 || b->num_seqs > (1 << 20) || b->num_tokens < 0 || b->num_tokens > (1 << 28))
    FAIL(Q3T_INVALID_INPUT, "%s: num_seqs %d outside 0..2^20 or num_tokens %d outside 0..2^28", what, b->num_seqs,
         b->num_tokens);
  if (b->max_q_len < 0 || b->max_kv_len < 0)
    FAIL(Q3T_INVALID_INPUT, "%s: negative max_q_len or max_kv_len", what);
  if (b->num_seqs > 0 && (!b->q_start || !b->kv_len)) FAIL(Q3T_INVALID_INPUT, "%s: null q_start or kv_len", what);
  if (!aligned(b->q_start, 4) || !aligned(b->kv_len, 4) || !aligned(b->table_row, 4))
    FAIL(Q3T_INVALID_INPUT, "%s: q_start, kv_len or table_row is not aligned to its entries", what);
  return Kv4Batch{b->num_seqs, b->num_tokens, b->q_start, b->kv_len, b->table_row, 0};
}

// Rows of `heads` heads: non-null, on an element boundary, no two overlapping.
void check_rows(const char *what, const char *name, const void *p, int64_t stride, int heads, int head_dim, int size) {
  if (!p) FAIL(Q3T_INVALID_INPUT, "%s: null %s rows", what, name);
  if (!aligned(p, size)) FAIL(Q3T_INVALID_INPUT, "%s: %s rows are not aligned to their element", what, name);
  if (stride < (int64_t)heads * head_dim)
    FAIL(Q3T_INVALID_INPUT, "%s: %s row stride %lld is below the row's %lld elements", what, name, (long long)stride,
         (long long)heads * head_dim);
}
bool wide(const void *p, int64_t stride, int size, int elems) {
  return !p || (aligned(p, (size_t)size * elems) && stride % elems == 0);
}

void rope_freqs(const char *what, const q3t_rope *r, double *freqs) {
  const int rot = r->rotary_dim;
  if (rot < 0 || rot > kKv4MaxDim || rot % 8)
    FAIL(Q3T_INVALID_INPUT, "%s: rotary_dim %d (a multiple of 8 up to %d)", what, rot, kKv4MaxDim);
  if (r->layout != Q3T_ROPE_HALF && r->layout != Q3T_ROPE_INTERLEAVED)
    FAIL(Q3T_INVALID_INPUT, "%s: unknown rotary layout %d", what, r->layout);
  if (r->scaling < Q3T_ROPE_NONE || r->scaling > Q3T_ROPE_BANDS)
    FAIL(Q3T_INVALID_INPUT, "%s: unknown rotary scaling %d", what, r->scaling);
  if (!(r->theta > 0.f) || !std::isfinite(r->theta) || !std::isfinite(r->amplitude))
    FAIL(Q3T_INVALID_INPUT, "%s: theta must be positive and theta and amplitude finite", what);
  if (r->scaling != Q3T_ROPE_NONE && (!(r->factor > 0.f) || !std::isfinite(r->factor)))
    FAIL(Q3T_INVALID_INPUT, "%s: rotary scaling needs a positive factor", what);
  if (r->scaling == Q3T_ROPE_BANDS && (!(r->low < r->high) || !std::isfinite(r->low) || !std::isfinite(r->high) ||
                                       r->original < 1))
    FAIL(Q3T_INVALID_INPUT, "%s: band scaling needs low < high and original > 0", what);
  for (int i = 0; i < rot / 2; i++) {
    // (64 powers are 2 us of an append's host time; theta^(2 / rot) multiplied up, even in 80 bits, gives other last
    // bits than the formula, and at far positions now and then another digit)
    double f = std::pow((double)r->theta, -2.0 * i / rot);
    if (r->scaling == Q3T_ROPE_LINEAR) f /= r->factor;
    if (r->scaling == Q3T_ROPE_BANDS) {
      const double turns = r->original * f / (2.0 * M_PI);
      const double keep = std::min(1.0, std::max(0.0, (turns - r->low) / ((double)r->high - r->low)));
      f = (1.0 - keep) * f / r->factor + keep * f;
    }
    freqs[i] = f;
  }
}

}  // namespace

extern "C" q3t_status q3t_rope_freqs(const q3t_rope *rope, double *freqs) {
  return guarded([&] {
    if (!rope || !freqs) FAIL(Q3T_INVALID_INPUT, "q3t_rope_freqs: null argument");
    double f[kKv4MaxDim / 2];
    rope_freqs("q3t_rope_freqs", rope, f);
    for (int i = 0; i < rope->rotary_dim / 2; i++) freqs[i] = f[i];
  });
}

extern "C" q3t_status q3t_kv4_append(const q3t_kv4_cache *cache, const q3t_kv4_batch *batch, const q3t_kv4_rows *rows,
                                     const q3t_rope *rope, void *stream) {
  const char *what = "q3t_kv4_append";
  return guarded([&] {
    Kv4AppendArgs a{};
    a.c = view_of(what, cache);
    a.b = batch_of(what, batch);
    if (!rows) FAIL(Q3T_INVALID_INPUT, "%s: null rows", what);
    if (rows->dtype != Q3T_F32 && rows->dtype != Q3T_BF16) FAIL(Q3T_INVALID_INPUT, "%s: unknown dtype %d", what, rows->dtype);
    if (rows->num_heads < 0 || rows->num_heads > (1 << 16))
      FAIL(Q3T_INVALID_INPUT, "%s: num_heads %d outside 0..65536", what, rows->num_heads);
    if (!aligned(rows->q_gamma, 4) || !aligned(rows->k_gamma, 4))
      FAIL(Q3T_INVALID_INPUT, "%s: q_gamma or k_gamma is not aligned to its elements", what);
    if (rope && rope->rotary_dim > a.c.head_dim)
      FAIL(Q3T_INVALID_INPUT, "%s: rotary_dim %d exceeds head_dim %d", what, rope->rotary_dim, a.c.head_dim);
    if ((rows->q_gamma || rows->k_gamma) && !(rows->eps >= 0.f && std::isfinite(rows->eps)))
      FAIL(Q3T_INVALID_INPUT, "%s: eps must be finite and not negative", what);
    if (rope) {
      rope_freqs(what, rope, a.rope.freq_pi);
      a.rope.rot = rope->rotary_dim;
      a.rope.interleaved = rope->layout == Q3T_ROPE_INTERLEAVED;
      a.rope.amplitude = rope->amplitude;
      for (int i = 0; i < a.rope.rot / 2; i++) a.rope.freq_pi[i] /= M_PI;
    }
    if (a.b.num_seqs == 0 || a.b.num_tokens == 0) return;
    const int D = a.c.head_dim, size = rows->dtype == Q3T_F32 ? 4 : 2;
    check_rows(what, "k", rows->k, rows->k_stride, a.c.n_kv, D, size);
    check_rows(what, "v", rows->v, rows->v_stride, a.c.n_kv, D, size);
    a.vec = wide(rows->k, rows->k_stride, size, 16 / size) && wide(rows->v, rows->v_stride, size, 16 / size);
    if (rows->num_heads) {
      check_rows(what, "q", rows->q, rows->q_stride, rows->num_heads, D, size);
      check_rows(what, "q_out", rows->q_out, rows->q_out_stride, rows->num_heads, D, 2);
      a.vec = a.vec && wide(rows->q, rows->q_stride, size, 16 / size) && wide(rows->q_out, rows->q_out_stride, 2, 8);
    }
    a.n_heads = rows->num_heads;
    a.q = rows->q, a.k = rows->k, a.v = rows->v;
    a.ldq = rows->q_stride, a.ldk = rows->k_stride, a.ldv = rows->v_stride;
    a.q_gamma = rows->num_heads ? rows->q_gamma : nullptr;
    a.k_gamma = rows->k_gamma;
    a.eps = rows->eps;
    a.q_out = (uint16_t *)rows->q_out;
    a.ldqo = rows->q_out_stride;
    DeviceScope dev(cache->device);
    CK(kv4_append(a, rows->dtype == Q3T_F32, (cudaStream_t)stream, true));
  });
}

extern "C" q3t_status q3t_kv4_attend(const q3t_kv4_cache *cache, const q3t_kv4_batch *batch, int num_heads,
                                     const uint16_t *q, int64_t q_stride, float scale, int window, uint16_t *out,
                                     int64_t out_stride, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *what = "q3t_kv4_attend";
  return guarded([&] {
    Kv4AttendArgs a{};
    a.c = view_of(what, cache);
    a.b = batch_of(what, batch);
    if (num_heads < 1 || num_heads > (1 << 16) || num_heads % a.c.n_kv)
      FAIL(Q3T_INVALID_INPUT, "%s: num_heads %d is not a multiple of the %d kv heads within 65536", what, num_heads,
           a.c.n_kv);
    if (!(std::fabs(scale) <= 0x1p127f)) FAIL(Q3T_INVALID_INPUT, "%s: scale %g is not within 2^127", what, (double)scale);
    if (window < 0) FAIL(Q3T_INVALID_INPUT, "%s: negative window", what);
    if (a.b.num_seqs == 0 || a.b.num_tokens == 0) return;
    check_rows(what, "q", q, q_stride, num_heads, a.c.head_dim, 2);
    check_rows(what, "out", out, out_stride, num_heads, a.c.head_dim, 2);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < (64 << 10))
      FAIL(Q3T_INVALID_INPUT, "%s: a workspace of 64 KiB at least on a 16-byte boundary is needed", what);
    a.n_heads = num_heads;
    a.q = q;
    a.ldq = q_stride;
    a.out = out;
    a.ldo = out_stride;
    a.scale = (float)((double)scale * M_LOG2E);
    a.window = window;
    a.vec = wide(q, q_stride, 2, 8) && wide(out, out_stride, 2, 8);
    DeviceScope dev(cache->device);
    CK(kv4_attend(a, batch->max_q_len, batch->max_kv_len, workspace, workspace_bytes, (cudaStream_t)stream, true));
  });
}

extern "C" q3t_status q3t_kv4_read(const q3t_kv4_cache *cache, const q3t_kv4_batch *batch, uint16_t *k, int64_t k_stride,
                                   uint16_t *v, int64_t v_stride, void *stream) {
  const char *what = "q3t_kv4_read";
  return guarded([&] {
    Kv4ReadArgs a{};
    a.c = view_of(what, cache);
    a.b = batch_of(what, batch);
    if (a.b.num_seqs == 0 || a.b.num_tokens == 0) return;
    if (!k && !v) FAIL(Q3T_INVALID_INPUT, "%s: neither k nor v rows", what);
    if (k) check_rows(what, "k", k, k_stride, a.c.n_kv, a.c.head_dim, 2);
    if (v) check_rows(what, "v", v, v_stride, a.c.n_kv, a.c.head_dim, 2);
    a.k = k, a.v = v;
    a.ldk = k_stride, a.ldv = v_stride;
    a.vec = wide(k, k_stride, 2, 8) && wide(v, v_stride, 2, 8);
    DeviceScope dev(cache->device);
    CK(kv4_read(a, (cudaStream_t)stream, true));
  });
}
