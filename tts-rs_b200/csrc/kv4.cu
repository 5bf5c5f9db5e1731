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

namespace q3t {

namespace {

// ---------------------------------------------------------------------------
// Which rows a CTA works on
// ---------------------------------------------------------------------------
// Token rows [t0, t0 + n) of sequence s, clamped to the call's rows; the
// last sits at position kv_len - 1.
Q3T_DEV void seq_rows(const Kv4Batch &b, int s, int &t0, int &n, int &pos0) {
  const int lo = min(max(b.q_start[s], 0), b.num_tokens), hi = min(max(b.q_start[s + 1], lo), b.num_tokens);
  t0 = lo;
  n = hi - lo;
  pos0 = b.kv_len[s] - n;
}

// Page of positions [16 p, 16 p + 16) of sequence s; -1 where the table or
// the pool has none.
Q3T_DEV int page_of(const Kv4View &c, const Kv4Batch &b, int s, int p) {
  const int row = b.table_row ? b.table_row[s] : s;
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
  const int first = max(pos0, w.p * 16), last = min(pos0 + n, w.p * 16 + 16);
  w.t0 = t0 + first - pos0;
  w.n = last - first;
  w.c0 = first - w.p * 16;
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
Q3T_DEV void load4(const float *p, bool vec, float v[4]) {
  if (vec) {
    const float4 u = *reinterpret_cast<const float4 *>(p);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = p[i];
  }
}
Q3T_DEV void load4(const uint16_t *p, bool vec, float v[4]) {
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    v[0] = bf2f(u.x & 0xffffu), v[1] = bf2f(u.x >> 16), v[2] = bf2f(u.y & 0xffffu), v[3] = bf2f(u.y >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = bf2f(p[i]);
  }
}
Q3T_DEV void store4(uint16_t *p, bool vec, const float v[4]) {
  if (vec) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = f2bf(v[i]);
  }
}

// RMSNorm of a row spread over LPR lanes, four dims each.  The sum of squares
// runs in 64 bits, so its order leaves no trace in the 32-bit factor.
template <int LPR>
Q3T_DEV void norm_row(float v[4], const float *gamma, float eps, int l) {
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 4; i++) ss += (double)v[i] * v[i];
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = (float)(1.0 / sqrt(ss / (4 * LPR) + (double)eps));
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = __fmul_rn(__fmul_rn(v[i], r), gamma[4 * l + i]);
}

// Rotation of a row by (cos, sin) per pair; every product and sum is rounded
// by itself, so a value does not depend on which of them a compiler fuses.
template <int LPR>
Q3T_DEV void rotate_row(float v[4], const float2 *cs, int rot, int interleaved, int l) {
  if (interleaved) {
    if (4 * l < rot) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float2 f = cs[2 * l + (i >> 1)];
        const float a = v[i], b = v[i + 1];
        v[i] = __fsub_rn(__fmul_rn(a, f.x), __fmul_rn(b, f.y));
        v[i + 1] = __fadd_rn(__fmul_rn(b, f.x), __fmul_rn(a, f.y));
      }
    }
    return;
  }
  const int q = rot >> 3;  // lanes of the first half (rot % 8 == 0)
  const bool first = l < q, in = l < 2 * q;
  const int src = first ? l + q : in ? l - q : l;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float p = __shfl_sync(0xffffffffu, v[i], src, LPR);
    if (in) {
      const float2 f = cs[4 * (first ? l : l - q) + i];
      const float a = __fmul_rn(v[i], f.x), b = __fmul_rn(p, f.y);
      v[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
  }
}

// Digits, scale and zero of the group of 32 that this lane's 8 lanes hold.  A
// group with a value that is not finite gets a NaN scale and zero: it reads
// back as NaN, as such a value does from a cache that is not quantised.
Q3T_DEV void quantise(const float v[4], uint32_t n[4], uint16_t &scale, uint16_t &zero) {
  float lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
  int bad = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) bad |= !(fabsf(v[i]) <= FLT_MAX);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad, o);
  }
  // towards minus infinity: more magnitude below zero, less above
  uint32_t zb = __float_as_uint(lo);
  zb = ((zb >> 31 && (zb << 1)) ? zb + 0xffffu : zb) & 0xffff0000u;
  if (zb == 0xff800000u) zb = 0xff7f0000u;
  const float z = __uint_as_float(zb);
  // halves first: the range of two finite values need not be finite
  const uint16_t sb = f2bf(__fmul_rn(__fsub_rn(__fmul_rn(hi, 0.5f), __fmul_rn(z, 0.5f)), (float)(2.0 / 15.0)));
  const float s = bf2f(sb);
  scale = bad ? 0x7fc0 : sb;
  zero = bad ? 0x7fc0 : (uint16_t)(zb >> 16);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float d = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v[i], z), s)), 0.f), 15.f);
    n[i] = !bad && s > 0.f ? (uint32_t)d : 0u;
  }
}

// ---------------------------------------------------------------------------
// Append: one CTA per (window, head split).  Rows go through a warp (D = 128)
// or half a warp (D = 64), four dims to a lane; blocks are put together in
// shared memory, and a window that fills its page is written in 16-byte
// pieces, any other in the bytes that its tokens own.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) k_kv4_append(const __grid_constant__ Kv4AppendArgs a) {
  constexpr int LPR = D / 4, RPW = 32 / LPR, G = D / 32, BLK = kv4_block_bytes(D);
  extern __shared__ __align__(16) uint8_t img[];  // [kv heads of this split][BLK]
  __shared__ float2 cs[kKv4Page][D / 2];
  pdl_wait();
  pdl_launch();
  Window w;
  if (!find_window(a.b, blockIdx.x, w) || w.p < 0) return;
  const int sp = a.splits, y = blockIdx.y;
  const int qh0 = (int)((int64_t)a.n_heads * y / sp), qh1 = (int)((int64_t)a.n_heads * (y + 1) / sp);
  const int kh0 = (int)((int64_t)a.c.n_kv * y / sp), kh1 = (int)((int64_t)a.c.n_kv * (y + 1) / sp);
  const int nq = qh1 - qh0, nk = kh1 - kh0;
  const int half = a.rope.rot / 2;
  for (int i = threadIdx.x; i < w.n * half; i += kAppendThreads) {
    const int c = i / half, f = i - c * half;
    double s, co;  // angles in 64 bits: a 32-bit product is off by its position's last bits
    sincospi((double)(w.p * 16 + w.c0 + c) * a.rope.freq_pi[f], &s, &co);
    cs[c][f] = make_float2((float)(co * a.rope.amplitude), (float)(s * a.rope.amplitude));
  }
  const int page = page_of(a.c, a.b, w.s, w.p);
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LPR, per = nq + 2 * nk, rows = w.n * per;
  for (int r0 = warp * RPW; r0 < rows; r0 += (kAppendThreads / 32) * RPW) {
    const int r = min(r0 + lane / LPR, rows - 1);  // a row past the end repeats the last one
    const int tok = r / per, hs = r - tok * per;
    const size_t row = (size_t)(w.t0 + tok);
    const int kind = hs < nq ? 0 : hs < nq + nk ? 1 : 2;
    const int head = kind == 0 ? qh0 + hs : kind == 1 ? kh0 + hs - nq : kh0 + hs - nq - nk;
    const T *src = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                   row * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + (size_t)head * D + 4 * l;
    float v[4];
    load4(src, a.vec, v);
    const float *gamma = kind == 0 ? a.q_gamma : kind == 1 ? a.k_gamma : nullptr;
    if (a.q_gamma || a.k_gamma) {  // the shuffles are for the whole warp
      float n[4] = {v[0], v[1], v[2], v[3]};
      norm_row<LPR>(n, gamma ? gamma : (a.q_gamma ? a.q_gamma : a.k_gamma), a.eps, l);
      if (gamma)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = n[i];
    }
    if (half) {
      float n[4] = {v[0], v[1], v[2], v[3]};
      rotate_row<LPR>(n, cs[tok], a.rope.rot, a.rope.interleaved, l);
      if (kind != 2)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = n[i];
    }
    uint32_t n[4];
    uint16_t scale, zero;
    quantise(v, n, scale, zero);
    if (kind == 0) store4(a.q_out + row * a.ldqo + (size_t)head * D + 4 * l, a.vec, v);
    // key bytes: b1 = 0, 1 of this lane's b0, the other b0 from the next lane;
    // value bytes: nibble h = 0 here, h = 1 two lanes on
    const uint32_t kb = n[0] | n[2] << 4 | n[1] << 16 | n[3] << 20, ko = __shfl_xor_sync(0xffffffffu, kb, 1);
    const uint32_t vn = n[0] | n[1] << 8 | n[2] << 16 | n[3] << 24, vo = __shfl_xor_sync(0xffffffffu, vn, 2);
    const int c = w.c0 + tok, t = (c >> 1) & 3;
    uint8_t *blk = img + (size_t)(head - kh0) * BLK;
    if (kind == 1 && !(l & 1))
      *reinterpret_cast<uint32_t *>(blk + c * (D / 2) + 4 * (G * ((l >> 1) & 3) + (l >> 3))) = kb | ko << 8;
    if (kind == 2 && !(l & 2)) {
      uint8_t *p = blk + 8 * D + 512 * (l >> 4) + 64 * (4 * (l & 1)) + 16 * t + 4 * ((l >> 2) & 3) + 2 * (c & 1) + (c >> 3);
#pragma unroll
      for (int i = 0; i < 4; i++) p[64 * i] = (uint8_t)((vn | vo << 4) >> 8 * i);
    }
    if (kind && !(l & 7)) {
      uint16_t *p = reinterpret_cast<uint16_t *>(blk + 16 * D + 8 * (4 * (4 * (l >> 3) + t) + 2 * (c >> 3) + (c & 1)));
      *reinterpret_cast<uint32_t *>(p + 2 * (kind - 1)) = scale | (uint32_t)zero << 16;
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
// and writes the rows n s + z, rounded once to bf16.
// ---------------------------------------------------------------------------
constexpr int kReadThreads = 256;

template <int D>
__global__ void __launch_bounds__(kReadThreads) k_kv4_read(const __grid_constant__ Kv4ReadArgs a) {
  constexpr int LPR = D / 4, RPC = kReadThreads / LPR, G = D / 32, BLK = kv4_block_bytes(D);
  extern __shared__ __align__(16) uint8_t img[];
  pdl_wait();
  pdl_launch();
  Window w;
  if (!find_window(a.b, blockIdx.x, w)) return;
  const int kh0 = (int)((int64_t)a.c.n_kv * blockIdx.y / a.splits);
  const int nk = (int)((int64_t)a.c.n_kv * (blockIdx.y + 1) / a.splits) - kh0;
  const int page = page_of(a.c, a.b, w.s, w.p);
  if (page >= 0) {
    const uint4 *src = reinterpret_cast<const uint4 *>(a.c.pool + ((size_t)page * a.c.n_kv + kh0) * BLK);
    for (int i = threadIdx.x; i < nk * (BLK / 16); i += kReadThreads) cp_async16(img + 16 * i, src + i, 16);
    cp_async_commit();
    cp_async_wait<0>();
  }
  __syncthreads();
  const int l = threadIdx.x % LPR;
  for (int r = threadIdx.x / LPR; r < 2 * nk * w.n; r += RPC) {
    const int is_v = r & 1, hc = r >> 1, tok = hc / nk, h = hc - tok * nk, c = w.c0 + tok, t = (c >> 1) & 3;
    uint16_t *out = is_v ? a.v : a.k;
    if (!out) continue;
    float x[4] = {0.f, 0.f, 0.f, 0.f};  // a position that has no page reads as zeros
    if (page >= 0) {
      const uint8_t *blk = img + (size_t)h * BLK;
      uint32_t n[4];
      if (!is_v) {
        const uint8_t *p = blk + c * (D / 2) + 4 * (G * ((l >> 1) & 3) + (l >> 3)) + (l & 1);
        n[0] = p[0] & 15, n[2] = p[0] >> 4, n[1] = p[2] & 15, n[3] = p[2] >> 4;
      } else {
        const uint8_t *p = blk + 8 * D + 512 * (l >> 4) + 64 * (4 * (l & 1)) + 16 * t + 4 * ((l >> 2) & 3) +
                           2 * (c & 1) + (c >> 3);
#pragma unroll
        for (int i = 0; i < 4; i++) n[i] = (p[64 * i] >> 2 * (l & 2)) & 15;
      }
      const uint32_t sz = *reinterpret_cast<const uint32_t *>(
          blk + 16 * D + 8 * (4 * (4 * (l >> 3) + t) + 2 * (c >> 3) + (c & 1)) + 4 * is_v);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = __fadd_rn(__fmul_rn((float)n[i], bf2f(sz & 0xffffu)), bf2f(sz >> 16));
    }
    store4(out + (size_t)(w.t0 + tok) * (is_v ? a.ldv : a.ldk) + (size_t)(kh0 + h) * D + 4 * l, a.vec, x);
  }
}

// ---------------------------------------------------------------------------
// Attend.  With q_d the query, per group j of 32 dims
//   score = sum_j [ s_j sum_{d in j} q_d n_d + z_j sum_{d in j} q_d ]
//   out_d = sum_keys (p s_j) n_d + sum_keys p z_j,  d in group j
// so the tensor cores see digits only, and scales and zeros enter once per
// (key, group).  The fragment rows are (query row r, group j): row (r, j) of
// the score product holds q in the dims of group j and zeros elsewhere, its
// accumulator is the group's share of the score, and the value product's
// column (r, j) holds p s_j.  Every lane then scales its own group's four
// keys of a page, two shuffles add the groups up, and the accumulators of
// both products meet without a transpose.
//
// A unit is (sequence, R query rows of one kv head), R = 8 NT / G; a cluster
// of CTAs shares a unit's pages, a warp takes two pages at a time through a
// cp.async ring, and the (m, l, o) parts of warps and CTAs are joined in
// order through shared and distributed shared memory: one launch, nothing
// kept between calls.
//
// f16 holds q times a power of two per row (its 11 bits keep a bf16 q whole
// down to 2^-25 of the row's largest) and p s times a power of two per warp,
// which follows the largest value scale: p s is rounded to 11 bits, as
// against the 8 of the output.  All sums, m and l are in 32 bits.
// ---------------------------------------------------------------------------
Q3T_DEV void mma_f16(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
Q3T_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 2^(14 - exponent of x), so that x times it lies in [2^14, 2^15)
Q3T_DEV float to_2p14(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 0xff);  // x >= 0
  const int f = min(max(127 + 14 + 127 - e, 1), 253);
  return __uint_as_float((uint32_t)f << 23);
}
Q3T_DEV float ld_cluster_f1(const float *p, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
// weight of a part with running maximum m and sum l under the joint maximum
// M; a part without keys has none, one with NaN scores keeps them
Q3T_DEV float part_weight(float m, float l, float M) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return exp2f(m - M);
}

constexpr int kAttendWarps = 4;

template <int D, int NT>
struct AttendCfg {
  static constexpr int G = D / 32, R = NT * 8 / G, BLK = kv4_block_bytes(D);
  static constexpr int NP = 2, ST = 3;  // pages of a step, steps in the ring
  static constexpr int RING = ST * NP * BLK;
  static constexpr size_t kSmem = (size_t)kAttendWarps * RING;
};

template <int D, int NT>
__global__ void __launch_bounds__(kAttendWarps * 32) k_kv4_attend(const __grid_constant__ Kv4AttendArgs a, int csize,
                                                                  int direct) {
  using Cfg = AttendCfg<D, NT>;
  constexpr int G = Cfg::G, R = Cfg::R, BLK = Cfg::BLK, NP = Cfg::NP, ST = Cfg::ST, W = kAttendWarps, MT = D / 16;
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ float s_m[W][R], s_l[W][R], s_z[W][R][G];
  __shared__ float c_m[R], c_l[R], c_o[R][D];
  pdl_wait();
  pdl_launch();
  const int rank = blockIdx.x % csize, unit = blockIdx.x / csize, kvh = unit % a.c.n_kv;
  const int gq = a.n_heads / a.c.n_kv;
  int s, tile;
  if (direct) {
    s = unit / a.c.n_kv;
    tile = 0;
  } else if (!find_item(
                 a.b.num_seqs, unit / a.c.n_kv,
                 [&](int q) {
                   int t0, n, pos0;
                   seq_rows(a.b, q, t0, n, pos0);
                   return (int)(((int64_t)n * gq + R - 1) / R);
                 },
                 s, tile)) {
    return;
  }
  int t0, n, pos0;
  seq_rows(a.b, s, t0, n, pos0);
  const int total = n * gq, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, j = g % G;
  uint8_t *ring = ring_all + warp * Cfg::RING;
  // a sequence with more rows than the caller announced takes more turns
  for (int row0 = tile * R; row0 < total; row0 += direct ? R : total) {
    const int nrow = min(R, total - row0);
    const int pos_lo = pos0 + row0 / gq, pos_hi = pos0 + (row0 + nrow - 1) / gq;
    const int key_lo = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
    const int pg_lo = key_lo >> 4, pg_hi = pos_hi < 0 ? pg_lo : (pos_hi >> 4) + 1;
    const int per = (max(pg_hi - pg_lo, 0) + csize - 1) / csize;
    const int p_beg = pg_lo + rank * per, p_end = min(p_beg + per, pg_hi);
    const int n_it = max(0, (p_end - p_beg - warp * NP + W * NP - 1) / (W * NP));

    // ---- queries ----
    uint32_t qa[NT][2][2];
    float qs[NT], sc[NT];
    int lim[NT], low[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = nt * (8 / G) + g / G, flat = min(row0 + r, total - 1);  // a row past the end repeats the last one
      const int tok = flat / gq, head = kvh * gq + flat - tok * gq;
      lim[nt] = pos0 + tok;
      low[nt] = a.window > 0 ? lim[nt] - a.window + 1 : 0;
      const uint16_t *qp = a.q + (size_t)(t0 + tok) * a.ldq + (size_t)head * D + 32 * j + 8 * t;
      float v[8];
      if (a.vec) {
        const uint4 u = *reinterpret_cast<const uint4 *>(qp);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = bf2f(x[i] & 0xffffu), v[2 * i + 1] = bf2f(x[i] >> 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = bf2f(qp[i]);
      }
      float top = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[i])), sum += v[i];
#pragma unroll
      for (int o = 1; o < 4 * G; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float f = to_2p14(top);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= f;
      // dims 0, 1 meet digits n 2^-24, dims 2, 3 meet 16 n 2^-24
      qa[nt][0][0] = pack_f16x2(v[0], v[1]);
      qa[nt][0][1] = pack_f16x2(v[2] * 0.0625f, v[3] * 0.0625f);
      qa[nt][1][0] = pack_f16x2(v[4], v[5]);
      qa[nt][1][1] = pack_f16x2(v[6] * 0.0625f, v[7] * 0.0625f);
      qs[nt] = sum * f * 0x1p-24f;
      sc[nt] = a.scale * 0x1p24f / f;
    }

    float m[NT], l[NT], zac[NT], acc[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      m[nt] = -INFINITY;
      l[nt] = zac[nt] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; i++) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
    }
    float vf = 1.f, vcap = 0.f;  // factor of the value scales, and the largest scale it is good for

    // ---- ring ----
    int ids = -1;           // pages of the next 32 / NP steps, by lane
    uint32_t has = 0;       // whether a page is there, the newest step in the low bits
    auto issue = [&](int it) {
      if (it < n_it) {
        if (it % (32 / NP) == 0) {
          const int p = p_beg + ((it + lane / NP) * W + warp) * NP + lane % NP;
          ids = p < p_end ? page_of(a.c, a.b, s, p) : -1;
        }
#pragma unroll
        for (int k = 0; k < NP; k++) {
          const int id = __shfl_sync(0xffffffffu, ids, (it % (32 / NP)) * NP + k);
          has = has << 1 | (id >= 0);
          if (id >= 0) {
            const uint8_t *src = a.c.pool + ((size_t)id * a.c.n_kv + kvh) * BLK;
            uint8_t *dst = ring + ((it % ST) * NP + k) * BLK;
#pragma unroll
            for (int i = 0; i < (BLK / 16 + 31) / 32; i++)
              if (BLK % 512 == 0 || lane + 32 * i < BLK / 16)
                cp_async16(dst + 16 * (lane + 32 * i), src + 16 * (lane + 32 * i), 16);
          }
        }
      } else {
        has <<= NP;
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) issue(i);
    for (int it = 0; it < n_it; it++) {
      issue(it + ST - 1);
      cp_async_wait<ST - 1>();
      __syncwarp();
      const int p0 = p_beg + (it * W + warp) * NP;
      const uint8_t *blk0 = ring + (it % ST) * NP * BLK;
      const uint32_t here = has >> ((ST - 1) * NP);  // bit NP - 1 - k: page k of this step
      // ---- scores of NP pages: y[nt][4 k + i], keys 2t, 2t+1, 2t+8, 2t+9 of page k ----
      float y[NT][4 * NP], vs[4 * NP], vz[4 * NP];
#pragma unroll
      for (int k = 0; k < NP; k++) {
        const uint8_t *blk = blk0 + k * BLK;
        float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w0[G], w1[G];
        if (G == 4) {
          const uint4 u = *reinterpret_cast<const uint4 *>(blk + g * (D / 2) + 4 * G * t);
          const uint4 x = *reinterpret_cast<const uint4 *>(blk + (g + 8) * (D / 2) + 4 * G * t);
          w0[0] = u.x, w0[1] = u.y, w0[G - 2] = u.z, w0[G - 1] = u.w;
          w1[0] = x.x, w1[1] = x.y, w1[G - 2] = x.z, w1[G - 1] = x.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2 *>(blk + g * (D / 2) + 4 * G * t);
          const uint2 x = *reinterpret_cast<const uint2 *>(blk + (g + 8) * (D / 2) + 4 * G * t);
          w0[0] = u.x, w0[1] = u.y, w1[0] = x.x, w1[1] = x.y;
        }
#pragma unroll
        for (int q = 0; q < G; q++) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t a0 = q == j ? qa[0][h][0] : 0u, a2 = q == j ? qa[0][h][1] : 0u;
            const uint32_t a1 = NT > 1 && q == j ? qa[NT - 1][h][0] : 0u, a3 = NT > 1 && q == j ? qa[NT - 1][h][1] : 0u;
            const uint32_t x0 = w0[q] >> 8 * h, x1 = w1[q] >> 8 * h;
            mma_f16(c0, a0, a1, a2, a3, x0 & 0x000f000fu, x0 & 0x00f000f0u);
            mma_f16(c1, a0, a1, a2, a3, x1 & 0x000f000fu, x1 & 0x00f000f0u);
          }
        }
        const uint4 *sp = reinterpret_cast<const uint4 *>(blk + 16 * D + 32 * (4 * j + t));
        const uint4 u0 = sp[0], u1 = sp[1];
        const uint32_t kw[4] = {u0.x, u0.z, u1.x, u1.z}, vw[4] = {u0.y, u0.w, u1.y, u1.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float ks = bf2f(kw[i] & 0xffffu), kz = bf2f(kw[i] >> 16);
          vs[4 * k + i] = bf2f(vw[i] & 0xffffu);
          vz[4 * k + i] = bf2f(vw[i] >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            const float c = i < 2 ? c0[2 * nt + i] : c1[2 * nt + i - 2];
            float x = fmaf(ks, c, kz * qs[nt]);
#pragma unroll
            for (int o = 4; o < 4 * G; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            y[nt][4 * k + i] = x * sc[nt];
          }
        }
        // keys that a row may not see, and pages that are not there: whatever
        // the slot holds, scales that are no numbers included, does not count
        const bool there = here >> (NP - 1 - k) & 1;
        const int key0 = (p0 + k) * 16;
        if (!there || key0 + 15 > pos_lo || (a.window > 0 && key0 < pos_hi - a.window + 1)) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int key = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
            bool any = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const bool seen = there && key <= lim[nt] && key >= low[nt];
              if (!seen) y[nt][4 * k + i] = -INFINITY;
              any |= seen;
            }
            if (!any) vs[4 * k + i] = vz[4 * k + i] = 0.f;
          }
        }
      }
      // ---- running maximum, factor of the value scales ----
      float top = 0.f, cr[NT];
#pragma unroll
      for (int i = 0; i < 4 * NP; i++) top = fmaxf(top, vs[i]);
      bool moved = top > vcap;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float mx = y[nt][0];
#pragma unroll
        for (int i = 1; i < 4 * NP; i++) mx = fmaxf(mx, y[nt][i]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[nt], mx);
        cr[nt] = m[nt] == mn ? 1.f : exp2f(m[nt] - mn);
        moved |= m[nt] != mn;
        m[nt] = mn;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float fv = 1.f;
        if (top > vcap) {
          const float nf = to_2p14(top);
          fv = nf * (1.f / vf);
          vf = nf;
          vcap = 0x1p15f / nf;
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          l[nt] *= cr[nt];
          zac[nt] *= cr[nt];
          // columns 2t and 2t + 1 belong to one row, that of lanes 4 (2t) ..
          const float f = __shfl_sync(0xffffffffu, cr[nt], 8 * t) * fv;
#pragma unroll
          for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[nt][i][e] *= f;
        }
      }
      // ---- p, p s and the value product ----
#pragma unroll
      for (int k = 0; k < NP; k++) {
        const uint8_t *blk = blk0 + k * BLK;
        uint32_t b0[NT], b1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const float mu = m[nt] == -INFINITY ? 0.f : m[nt];
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float yi = y[nt][4 * k + i], p = exp2f(yi - mu);
            const bool out = yi == -INFINITY;  // p is 0: its value may be anything
            l[nt] += p;
            zac[nt] += out ? 0.f : p * vz[4 * k + i];
            w[i] = out ? 0.f : p * (vs[4 * k + i] * vf);
          }
          b0[nt] = pack_f16x2(w[0], w[1]);
          b1[nt] = pack_f16x2(w[2], w[3]);
        }
#pragma unroll
        for (int M = 0; M < D / 64; M++) {
          const uint4 u = *reinterpret_cast<const uint4 *>(blk + 8 * D + 512 * M + 16 * lane);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t x = w[i], x8 = x >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              mma_f16(acc[nt][4 * M + i], x & 0x000f000fu, x & 0x00f000f0u, x8 & 0x000f000fu, x8 & 0x00f000f0u, b0[nt],
                      b1[nt]);
          }
        }
      }
      __syncwarp();  // every lane is done with the stage that the next copies write
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring is free: it takes the warps' parts
    float *s_o = reinterpret_cast<float *>(ring_all);  // [W][R][D]
    const float back = 1.f / vf;  // digits were n 2^-24 and 16 n 2^-24
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float lt = l[nt], zt = zac[nt];
      lt += __shfl_xor_sync(0xffffffffu, lt, 1);
      lt += __shfl_xor_sync(0xffffffffu, lt, 2);
      zt += __shfl_xor_sync(0xffffffffu, zt, 1);
      zt += __shfl_xor_sync(0xffffffffu, zt, 2);
      const int rg = nt * (8 / G) + g / G, rt = nt * (8 / G) + 2 * t / G;
      if (t == 0) {
        s_z[warp][rg][j] = zt;
        if (j == 0) {
          s_m[warp][rg] = m[nt];
          s_l[warp][rg] = lt;
        }
      }
      float *o = s_o + ((size_t)warp * R + rt) * D;
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          if ((2 * t + e) % G == i / 2) {
            o[16 * i + g] = acc[nt][i][e] * 0x1p24f * back;
            o[16 * i + 8 + g] = acc[nt][i][2 + e] * 0x1p20f * back;
          }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * D; i += W * 32) {
      const int r = i / D, d = i - r * D;
      float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < W; w++) M = fmaxf(M, s_m[w][r]);
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float f = part_weight(s_m[w][r], s_l[w][r], M);
        L += f * s_l[w][r];
        o += f * (s_o[((size_t)w * R + r) * D + d] + s_z[w][r][d / 32]);
      }
      c_o[r][d] = o;
      if (d == 0) {
        c_m[r] = M;
        c_l[r] = L;
      }
    }
    if (csize > 1)
      cluster_sync();
    else
      __syncthreads();
    if (rank == 0)
      for (int i = threadIdx.x; i < nrow * D; i += W * 32) {
        const int r = i / D, d = i - r * D, tok = (row0 + r) / gq, head = kvh * gq + (row0 + r) - tok * gq;
        float M = c_m[r], L = c_l[r], o = c_o[r][d];
        for (int k = 1; k < csize; k++) {
          const float mk = ld_cluster_f1(&c_m[r], k), lk = ld_cluster_f1(&c_l[r], k), ok = ld_cluster_f1(&c_o[r][d], k);
          const float Mn = fmaxf(M, mk), fa = part_weight(M, L, Mn), fb = part_weight(mk, lk, Mn);
          L = fa * L + fb * lk;
          o = fa * o + fb * ok;
          M = Mn;
        }
        a.out[(size_t)(t0 + tok) * a.ldo + (size_t)head * D + d] = f2bf(L == 0.f ? 0.f : o / L);  // no keys: zeros
      }
    if (csize > 1)
      cluster_sync();  // a CTA's part stays until rank 0 has read it
    else
      __syncthreads();
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

template <typename T, int D>
cudaError_t append_launch(const Kv4AppendArgs &a, int windows, cudaStream_t st, bool pdl) {
  static std::atomic<uint64_t> done{0};
  const int per = (a.c.n_kv + a.splits - 1) / a.splits;
  const size_t smem = (size_t)per * kv4_block_bytes(D);
  cudaError_t e = once_per_device(done, [] {
    return cudaFuncSetAttribute(k_kv4_append<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10);
  });
  if (e != cudaSuccess) return e;
  return launch(k_kv4_append<T, D>, dim3(windows, a.splits), kAppendThreads, smem, 1, pdl, st, a);
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
cudaError_t attend_launch(const Kv4AttendArgs &a, int max_q, int max_kv, cudaStream_t st, bool pdl) {
  using Cfg = AttendCfg<D, NT>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = once_per_device(done, [] {
    cudaError_t r = cudaFuncSetAttribute(k_kv4_attend<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Cfg::kSmem);
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(k_kv4_attend<D, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  const int gq = a.n_heads / a.c.n_kv;
  const bool direct = max_q > 0 && (int64_t)max_q * gq <= Cfg::R;
  int64_t tiles = direct ? a.b.num_seqs : ((int64_t)a.b.num_tokens * gq + Cfg::R - 1) / Cfg::R + a.b.num_seqs;
  const int64_t units = tiles * a.c.n_kv;
  // CTAs of a unit: enough to occupy the SMs, while each warp still gets two steps of pages
  const int pages = (a.window > 0 && (max_kv <= 0 || a.window < max_kv) ? a.window + 31 : max_kv > 0 ? max_kv : 4096) / 16 + 1;
  int c = 1;
  while (c < 16 && units * c < 296 && c * kAttendWarps * Cfg::NP * 2 < pages) c *= 2;
  if (units * c > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch(k_kv4_attend<D, NT>, dim3((unsigned)(units * c)), kAttendWarps * 32, Cfg::kSmem, c, pdl, st, a, c,
                direct ? 1 : 0);
}

}  // namespace

cudaError_t kv4_append(const Kv4AppendArgs &a0, bool f32_rows, cudaStream_t st, bool pdl) {
  const int windows = max_windows(a0.b);
  if (windows <= 0 || a0.b.num_seqs <= 0) return cudaSuccess;
  Kv4AppendArgs a = a0;
  a.splits = head_splits(windows, a.c.n_kv);
  // a split's blocks have to fit shared memory
  while ((size_t)((a.c.n_kv + a.splits - 1) / a.splits) * kv4_block_bytes(a.c.head_dim) > (40 << 10)) a.splits++;
  if (a.c.head_dim == 128)
    return f32_rows ? append_launch<float, 128>(a, windows, st, pdl) : append_launch<uint16_t, 128>(a, windows, st, pdl);
  return f32_rows ? append_launch<float, 64>(a, windows, st, pdl) : append_launch<uint16_t, 64>(a, windows, st, pdl);
}

cudaError_t kv4_read(const Kv4ReadArgs &a0, cudaStream_t st, bool pdl) {
  const int windows = max_windows(a0.b);
  if (windows <= 0 || a0.b.num_seqs <= 0) return cudaSuccess;
  Kv4ReadArgs a = a0;
  a.splits = head_splits(windows, a.c.n_kv);
  while ((size_t)((a.c.n_kv + a.splits - 1) / a.splits) * kv4_block_bytes(a.c.head_dim) > (40 << 10)) a.splits++;
  return a.c.head_dim == 128 ? read_launch<128>(a, windows, st, pdl) : read_launch<64>(a, windows, st, pdl);
}

cudaError_t kv4_attend(const Kv4AttendArgs &a, int max_q, int max_kv, cudaStream_t st, bool pdl) {
  if (a.b.num_tokens <= 0 || a.b.num_seqs <= 0) return cudaSuccess;
  const int rows = (max_q > 0 ? max_q : 2) * (a.n_heads / a.c.n_kv);  // rows of a kv head: one column tile, or two
  if (a.c.head_dim == 128)
    return rows <= 2 ? attend_launch<128, 1>(a, max_q, max_kv, st, pdl) : attend_launch<128, 2>(a, max_q, max_kv, st, pdl);
  return rows <= 4 ? attend_launch<64, 1>(a, max_q, max_kv, st, pdl) : attend_launch<64, 2>(a, max_q, max_kv, st, pdl);
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
  if (c->table_rows < 1 || c->table_stride < 1)
    FAIL(Q3T_INVALID_INPUT, "%s: page table of %d x %d", what, c->table_rows, c->table_stride);
  if (!c->pool || !c->page_table) FAIL(Q3T_INVALID_INPUT, "%s: null pool or page table", what);
  if (!aligned(c->pool, 16)) FAIL(Q3T_INVALID_INPUT, "%s: the pool must start on a 16-byte boundary", what);
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
  return Kv4Batch{b->num_seqs, b->num_tokens, b->q_start, b->kv_len, b->table_row};
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
    a.vec = wide(rows->k, rows->k_stride, size, 4) && wide(rows->v, rows->v_stride, size, 4);
    if (rows->num_heads) {
      check_rows(what, "q", rows->q, rows->q_stride, rows->num_heads, D, size);
      check_rows(what, "q_out", rows->q_out, rows->q_out_stride, rows->num_heads, D, 2);
      a.vec = a.vec && wide(rows->q, rows->q_stride, size, 4) && wide(rows->q_out, rows->q_out_stride, 2, 4);
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
                                     int64_t out_stride, void *stream) {
  const char *what = "q3t_kv4_attend";
  return guarded([&] {
    Kv4AttendArgs a{};
    a.c = view_of(what, cache);
    a.b = batch_of(what, batch);
    if (num_heads < 1 || num_heads > (1 << 16) || num_heads % a.c.n_kv)
      FAIL(Q3T_INVALID_INPUT, "%s: num_heads %d is not a multiple of the %d kv heads within 65536", what, num_heads,
           a.c.n_kv);
    if (!std::isfinite(scale)) FAIL(Q3T_INVALID_INPUT, "%s: scale must be finite", what);
    if (window < 0) FAIL(Q3T_INVALID_INPUT, "%s: negative window", what);
    if (a.b.num_seqs == 0 || a.b.num_tokens == 0) return;
    check_rows(what, "q", q, q_stride, num_heads, a.c.head_dim, 2);
    check_rows(what, "out", out, out_stride, num_heads, a.c.head_dim, 2);
    a.n_heads = num_heads;
    a.q = q;
    a.ldq = q_stride;
    a.out = out;
    a.ldo = out_stride;
    a.scale = (float)((double)scale * M_LOG2E);
    a.window = window;
    a.vec = wide(q, q_stride, 2, 8) && wide(out, out_stride, 2, 8);
    DeviceScope dev(cache->device);
    CK(kv4_attend(a, batch->max_q_len, batch->max_kv_len, (cudaStream_t)stream, true));
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
    a.vec = wide(k, k_stride, 2, 4) && wide(v, v_stride, 2, 4);
    DeviceScope dev(cache->device);
    CK(kv4_read(a, (cudaStream_t)stream, true));
  });
}
