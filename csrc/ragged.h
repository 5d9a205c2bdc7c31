// Argument structs and launchers of the ragged-batch operators: sequences of
// different lengths, packed one after another without padding, over a KV
// cache held in pages. These operators have no counterpart in the reference,
// whose batches are padded to one length.
//
// Page pool: k_pages, v_pages [num_pages, nkv, page_size, D]; position p of
// sequence b lies in page page_table[b][p / page_size] at row p % page_size.
// page_size is a multiple of 16. Element type bf16 or fp16, D 64 or 128.
//
// Index data (page ids, lengths, offsets) lives on the device and is checked
// there: an entry out of range is recorded in `status` (kBoundsViolation)
// and never dereferenced (each struct says what is computed instead).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace afd {

enum ElemType : int { kElemBf16 = 0, kElemF16 = 1, kElemF32 = 2 };

// Attention of one new token per sequence: query b sees positions
// 0 .. seq_lens[b] - 1. A length of zero gives zeros; so does, with a record
// in `status`, one outside [0, max_pages * page_size]. A page id outside
// [0, num_pages) is recorded and its keys and values read as zeros.
struct PagedDecodeArgs {
  const void* q;            // [B, nq, D], rows q_row elements apart
  long long q_row;
  const void* k_pages;
  const void* v_pages;
  long long page_stride;    // elements between pages
  const int* page_table;    // [B, max_pages], rows table_row ints apart
  int table_row;
  const int* seq_lens;      // [B]
  void* out;                // [B, nq, D]
  int B, nq, nkv, D, num_pages, page_size, max_pages;
  float scale;              // > 0
  int elem;
  int* status;              // optional [2]
  void* parts;              // [paged_decode_part_bytes], 16-byte aligned
  int* counters;            // [paged_decode_counters], zero; left zero
};
// Workspace of a launch.
long long paged_decode_part_bytes(int nq, int nkv, int D, int num_sms);
int paged_decode_counters(int num_sms);
int launch_paged_decode(const PagedDecodeArgs& a, int num_sms, cudaStream_t s);

// Causal attention of packed queries. Sequence i owns query rows
// cu_q[i] .. cu_q[i+1] - 1; they are its last positions. Keys and values come
// packed (k, v, cu_k: key rows of the sequences) or from pages (seq_lens: all
// positions, the new ones included). A query whose position is negative
// (more queries than keys) sees no key and gets zeros, and so do rows before
// cu_q[0] and past cu_q[n]. Offsets outside [0, rows] are clamped and recorded; with
// query offsets that still decrease then, which is recorded too, all rows get zeros,
// and with key offsets that do, the sequence has no key. Lengths and page ids as in
// PagedDecodeArgs. A call without rows of queries, or of keys, checks no offset.
struct PackedAttnArgs {
  const void* q;            // [T, nq, D], rows q_row elements apart
  long long q_row;
  int T;
  const int* cu_q;          // [n + 1]
  int n_seqs;
  const void* k;            // packed [Tk, nkv, D], rows k_row elements apart
  const void* v;
  long long k_row, v_row;
  int Tk;
  const int* cu_k;          // [n + 1]
  int paged;                // keys and values from the pool instead
  const void* k_pages;
  const void* v_pages;
  long long page_stride;
  const int* page_table;    // [n, max_pages]
  int table_row;
  const int* seq_lens;      // [n]
  int num_pages, page_size, max_pages;
  void* out;                // [T, nq, D]
  int nq, nkv, D;
  float scale;              // > 0
  int elem;
  int* status;
  int* counter;             // [1], zero; left zero
  int splits;               // parts of a block's keys at most; 1: none is split
  float* part_o;            // filled in by the launch: O [splits, T, nq, D],
  float2* part_ml;          // largest score and sum [splits, T, nq],
  int* n_parts;             // parts [T, nq]
};
// Parts that fill the GPU where there are few blocks, for keys up to most_keys.
int packed_attention_splits(long long T, int n_seqs, int nq, int nkv, long long most_keys,
                            int num_sms);
long long packed_attention_part_bytes(long long rows, int D, int splits);
int launch_packed_attention(const PackedAttnArgs& a, void* parts, int num_sms, cudaStream_t s);

// Per-head RMSNorm and RoPE of the q and k heads of a packed qkv projection.
// q goes to q_out; k to k_out [T, nkv, D], or with the pool given, k and v to
// the page rows slots[t] (= page * page_size + row; negative: not stored).
// A slot or position out of range is recorded; the row is then not stored, or
// the position clamped to the table.
struct NormRopeArgs {
  const void* qkv;          // [T, (nq + 2 nkv) D], rows qkv_row elements apart
  long long qkv_row;
  const void* q_norm;       // [D]
  const void* k_norm;
  const float* rope;        // [max_pos, D]: cos | sin
  int max_pos;
  const int* positions;     // [T]
  const int64_t* slots;     // [T], with the pool
  void* q_out;              // [T, nq, D]
  void* k_out;              // [T, nkv, D], without the pool
  void* k_pages;            // nullptr: no pool
  void* v_pages;
  long long page_stride;
  int num_pages, page_size;
  int T, nq, nkv, D;
  float eps;
  int elem;
  int* status;
};
int launch_norm_rope(const NormRopeArgs& a, cudaStream_t s);

// Log-probability of ids[r], entropy of the row, and the top_k logits of the
// row (larger first, equal ones by index).
struct TokenLogprobsArgs {
  const void* logits;       // [R, V], rows `row` elements apart
  long long row;
  const int64_t* ids;       // [R]; an id outside [0, V) gives NaN
  float* logprob;           // [R]
  float* entropy;           // [R]
  int64_t* top_ids;         // [R, top_k]
  float* top_logprobs;      // [R, top_k]
  int R, V, top_k;          // V <= kMaxLogprobVocab, top_k <= kMaxTopLogprobs
  int elem;
  int* counters;            // with splits > 1: [R], zero; left zero
  float* parts;             // set by the launcher
  float* block_max;
};
constexpr int kMaxTopLogprobs = 32;
constexpr int kMaxLogprobVocab = 1 << 21;
// CTAs per row, the bytes of workspace for them (16-byte aligned), the launch.
int token_logprobs_splits(int R, int V, int num_sms);
long long token_logprobs_workspace(int R, int V, int splits);
int launch_token_logprobs(const TokenLogprobsArgs& a, int splits, void* ws, cudaStream_t s);

}  // namespace afd
