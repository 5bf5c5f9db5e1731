// 4-bit paged key/value cache: device views and launchers of the operators
// (kv4.cu), shared by the C ABI and the decode engine.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace q3t {

constexpr int kKv4Page = 16;    // tokens of a page
constexpr int kKv4Group = 32;   // dims that share a scale and a zero
constexpr int kKv4MaxDim = 128;

// Bytes of one (page, kv head) block: 8 D key digits, 8 D value digits, 4 D
// scales (see q3t_kv4_cache in q3t.h for the order inside).
constexpr int kv4_block_bytes(int head_dim) { return 20 * head_dim; }

// One layer's blocks and the page table.
struct Kv4View {
  uint8_t *pool;          // [num_pages][n_kv][block]
  const int *table;       // [table_rows][table_stride]
  int64_t num_pages;
  int n_kv, head_dim, table_rows, table_stride;
};

// The token rows of a call, by sequence (device arrays).
struct Kv4Batch {
  int num_seqs, num_tokens;
  const int *q_start;   // [num_seqs + 1]
  const int *kv_len;    // [num_seqs]
  const int *table_row; // [num_seqs], nullable: then row first + s
  int first;
};

// Rotation of the leading `rot` dims: freq[i] = radians per position / pi.
struct Kv4Rope {
  int rot;          // 0: none
  int interleaved;  // pairs (2i, 2i + 1) instead of (i, i + rot / 2)
  float amplitude;
  double freq_pi[kKv4MaxDim / 2];
};

struct Kv4AppendArgs {
  Kv4View c;
  Kv4Batch b;
  Kv4Rope rope;
  int n_heads;            // query heads (0: none)
  const void *q, *k, *v;  // rows, f32 or bf16
  int64_t ldq, ldk, ldv;  // elements between token rows
  const float *q_gamma, *k_gamma;  // nullable
  float eps;
  uint16_t *q_out;        // bf16 rows
  int64_t ldqo;
  int vec;                // every row starts on a 16-byte boundary
  int splits;             // head splits (gridDim.y)
};

struct Kv4AttendArgs {
  Kv4View c;
  Kv4Batch b;
  int n_heads;
  const uint16_t *q;  // bf16 rows
  int64_t ldq;
  uint16_t *out;
  int64_t ldo;
  float scale;        // of the scores, times log2(e)
  int window;         // keys a query sees at most (0: all before it)
  int vec;            // q and out rows start on 16-byte boundaries
  int *err;           // set (bitwise or) when a bounded wait gave up; nullable
  int big;            // launcher: sequences of more rows are another kernel's (0: none)
  int units;          // launcher: units of a few rows that a sequence has, as far as announced
};

struct Kv4ReadArgs {
  Kv4View c;
  Kv4Batch b;
  uint16_t *k, *v;    // bf16 rows, nullable
  int64_t ldk, ldv;
  int vec;            // every row starts on a 16-byte boundary
  int splits;
};

// Append and attend of one layer of a talker pass.
struct Kv4Step {
  Kv4AppendArgs append;
  Kv4AttendArgs attend;
  int max_q, max_kv;
  void *ws;  // kKv4Workspace bytes
};

// max_q / max_kv: the most tokens and keys of a sequence, as the caller knows
// them; they choose the launch shape only (0: unknown).  Launch errors are
// returned; `pdl` lets the launch overlap the tail of the one before it.
cudaError_t kv4_append(const Kv4AppendArgs &a, bool f32_rows, cudaStream_t st, bool pdl);
// attend needs a workspace: 64 KiB at least, kKv4Workspace for the widest launch.
constexpr int64_t kKv4Workspace = 20 << 20;
cudaError_t kv4_attend(const Kv4AttendArgs &a, int max_q, int max_kv, void *ws, int64_t ws_bytes, cudaStream_t st,
                       bool pdl);
cudaError_t kv4_read(const Kv4ReadArgs &a, cudaStream_t st, bool pdl);

}  // namespace q3t
