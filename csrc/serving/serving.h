// Operators of one token step of a served language model (gfx950).
//
// Every launch_* function checks nothing that its caller can check on the
// host, enqueues on `stream`, allocates nothing, keeps nothing and never
// throws; it returns the launch's hipError_t. Workspaces are the caller's.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace serving {

enum DType : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

// ---- product with 4-bit weights -------------------------------------------
struct W4Args {
  const void* x;          // [m, k], rows ldx elements apart
  const uint8_t* codes;   // [ceil(n/16)][ceil(k/128)][64][16]
  const void* scales;     // [ceil(n/16)][groups][16], x's type
  const uint8_t* zeros;   // like scales, or null: every zero point is 8
  void* y;                // [m, n], rows ldy elements apart
  int64_t ldx, ldy;
  int m, n, k, group;     // group: 32, 64 or 128
  int dtype;              // kBF16 or kF16
  void* work;             // w4_workspace() bytes, or null if 0
};
int64_t w4_workspace(const W4Args& a);
// Largest K: its scales and zero points have to fit the LDS.
constexpr int kMaxColumns = 32768;
constexpr int kMaxTokens = 65472;  // a grid's second dimension, in whole chunks
hipError_t launch_w4_matmul(const W4Args& a, hipStream_t stream);

// ---- 8-bit paged cache ----------------------------------------------------
struct CacheArgs {
  uint8_t* k;             // e4m3 [pages][heads][page][dim]
  uint8_t* v;             // e4m3 [pages][heads][dim][page]
  float* k_scale;         // [pages][heads]
  float* v_scale;
  const int32_t* table;   // [batch][blocks], rows ldt apart
  const int32_t* lens;    // [batch] tokens held, the new ones included
  const int32_t* starts;  // [batch + 1] first row of each sequence, or null:
                          // row b is sequence b's only one
  int64_t ldt;
  int pages, heads, page, dim, batch, blocks;
  int rows;               // query or new tokens in all
};

struct AppendArgs {
  CacheArgs c;
  const void* k_new;      // [rows][heads][dim], last dimension dense
  const void* v_new;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  int dtype;
};
hipError_t launch_cache_append(const AppendArgs& a, hipStream_t stream);

// Rows behind the last sequence: left alone; their lse becomes -inf; their
// output becomes 0 as well.
enum Tail : int { kLeaveTail = 0, kTailLse = 1, kFillTail = 2 };

struct AttentionArgs {
  CacheArgs c;
  const void* q;          // [rows][q_heads][dim], last dimension dense
  void* out;              // [rows][q_heads][dim], last dimension dense
  float* lse;             // [rows][q_heads]
  float* work;            // plan_attention() floats, or null if 0
  int64_t q_row, q_head, o_row, o_head;
  int q_heads, window;    // window 0: none
  int tail;               // a Tail: what becomes of rows behind the last sequence
  float scale;
  int dtype;
  int64_t longest;        // longest sequence as far as known: steers the split
  // of a pass, by plan_attention()
  int splits, chunk;      // workgroups of a context, and the tokens of one
  int row_tile;           // rows (token, head) of a workgroup
  int per;                // tiles of a sequence, 0: as many as its rows need
  int few, many;          // takes the sequences with more than few, at most many rows
};
// Sequences with few rows and those with many take passes of their own.
struct AttentionPlan {
  AttentionArgs pass[2];
  int passes;
  int64_t floats;         // of workspace
};
AttentionPlan plan_attention(const AttentionArgs& a);
hipError_t launch_cache_attention(const AttentionArgs& a, hipStream_t stream);

// ---- log probabilities of given tokens ------------------------------------
struct LogprobArgs {
  const void* logits;     // [rows][vocab], rows ld elements apart
  const int64_t* targets; // [rows]
  float* logprob;         // [rows]
  float* entropy;         // [rows]
  int64_t* rank;          // [rows]
  int64_t* top_ids;       // [rows][top] or null
  float* top_logprobs;
  float* work;            // logprob_workspace() floats
  int64_t ld;
  int64_t rows;
  int vocab, top, dtype;
};
int64_t logprob_workspace(int64_t rows, int vocab, int dtype);
hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream);

constexpr int kMaxTop = 64;
constexpr int kMaxVocab = 1 << 22;

}  // namespace serving
