// Host side of the sequence operators: rotary positions, paged key/value cache, attention over
// it and over ragged rows.  Parameter blocks are fully checked by the C ABI (seq_api.cpp)
// before a launch; what only the device knows (lengths, page numbers) the kernels check.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace ivh {

enum SeqType : int { kSeqF16 = 0, kSeqBF16 = 1, kSeqF32 = 2 };  // the last: logits alone

// Rotation of a head's leading `rot` channels by positions with up to four axes.
struct RotParams {
  int rot = 0, half = 0;      // rotated channels (0: none), rot / 2 frequencies
  int axes = 1;
  int sec[4] = {0, 0, 0, 0};  // frequencies of each axis
  int adjacent = 0;           // pairs (2i, 2i + 1), else (i, i + half)
  int dealt = 0;              // axes in turn, else one section after the other
  const int32_t * pos = nullptr;
  long pos_axis = 0;
  const float * freq = nullptr;
};

struct RopeParams {
  RotParams r;
  int type = 0, heads = 0, dim = 0;
  long tokens = 0;
  const void * x = nullptr;
  void * y = nullptr;
  long x_token = 0, x_head = 0, y_token = 0, y_head = 0;
};
void launch_rope(const RopeParams & p, hipStream_t s);

// A paged cache: kc [pages][heads][page / 4][dim / E][4][E], vc [pages][heads][page / E][dim][E]
// with E = 16 bytes' worth of elements; ks, vs [pages][heads] for 8-bit pages.
struct CacheParams {
  int type = 0, bits = 8, heads = 0, dim = 0, page = 0, pages = 0, width = 0;
  void * kc = nullptr;
  void * vc = nullptr;
  float * ks = nullptr;
  float * vs = nullptr;
  const int32_t * table = nullptr;  // [batch][width]
  const int32_t * cu = nullptr;     // [batch + 1]
  const int32_t * lens = nullptr;   // [batch], with the new tokens
  int batch = 0, tokens = 0;
};

struct AppendParams {
  CacheParams c;
  RotParams r;
  const void * k = nullptr;
  const void * v = nullptr;
  long k_token = 0, k_head = 0, v_token = 0, v_head = 0;
};
void launch_kv_append(const AppendParams & p, hipStream_t s);

struct PagedParams {
  CacheParams c;
  const void * q = nullptr;
  void * o = nullptr;
  long q_token = 0, q_head = 0, o_token = 0, o_head = 0;
  int heads = 0, group = 1;      // query heads, and those that share a key head
  float scale_log2 = 1.0f;       // softmax scale times log2 e
  int window = 0, sinks = 0;     // window 0: every earlier key
  // how a call is split, from paged_split
  int row_tiles = 1;             // 16-row tiles of a work-group
  int row_waves = 1;             // waves that take rows; the others of four share a row's keys
  int row_slots = 1;             // work-groups over the rows of a sequence and key head
  int parts = 1, part_steps = 1; // work-groups over the keys, and 64-key steps of each at least
  float * ws = nullptr;          // parts > 1: partial sums [parts][tokens][heads][dim], maxima and sums
  // with shared first tokens: each sequence's own keys have parts `lead` .. all_parts - 1 of the workspace
  const int32_t * member = nullptr;  // [groups + 1] first sequences
  const int32_t * shared = nullptr;  // [groups] tokens
  int groups = 0, lead = 0, all_parts = 1;
  int shared_wgs = 0, shared_slots = 1, shared_steps = 1;  // both kinds of keys in one launch: the split of the shared ones
};
// Sets the split of a call with at most max_new new tokens and max_len cached ones in a
// sequence (bounds that only steer the split); returns the workspace bytes.
size_t paged_split(PagedParams & p, int max_new, int max_len);
// Work-groups of 256 lanes over the keys of `seqs` sequences or groups.  A launch holds fewer than 2^24.
long paged_wgs(const PagedParams & p, long seqs);
// Rows are joined `per` a work-group, by `lots` lots of lanes each, in launches of at most kJoinWgs (a millisecond's work).
struct JoinSplit {
  int lots, per;
  long wgs;
};
constexpr long kJoinWgs = 1L << 20;
JoinSplit join_split(const PagedParams & p);
void launch_paged_attention(const PagedParams & p, hipStream_t s);
void launch_paged_bf16(const PagedParams & p, hipStream_t s);  // its bf16 kernels, built by themselves

// Attention with shared first tokens: the split of both kinds of keys, those of groups first.
struct PrefixParams {
  PagedParams first, own;
  int many = 0;  // shared keys by work-groups of 128 rows
  int both = 0;  // both kinds of keys in one launch,
  int wide = 0;  // shared ones for 32 rows at a time, else as the paged attention does
};
size_t prefix_split(PrefixParams & p, int max_new, int max_len, int max_shared);
void launch_prefix_attention(const PrefixParams & p, hipStream_t s);
void launch_prefix_bf16(const PrefixParams & p, hipStream_t s);

struct LinearParams {
  int type = 0, heads = 0, group = 1, key_dim = 0, dim = 0;  // group: heads that share queries and keys
  int batch = 0, tokens = 0, slots = 0;
  float scale = 1.0f;
  const void * q = nullptr;
  const void * k = nullptr;
  const void * v = nullptr;
  const float * g = nullptr;
  const int32_t * cu = nullptr;
  const int32_t * from = nullptr;
  const int32_t * to = nullptr;
  float * state = nullptr;
  void * o = nullptr;
  long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0, o_token = 0, o_head = 0, g_token = 0, g_head = 0;
  // how a call is split, from linear_split
  int seg = 0;                   // tokens of a segment, 0: token by token
  float * ws = nullptr;          // first states of segments [tokens / seg + batch][heads][key_dim][dim], null: one each
  float * decay = nullptr;       // of whole segments, behind them: a number and a power of two for each
};
// Sets the split of a call with at most max_new rows in a sequence; returns the workspace bytes.
size_t linear_split(LinearParams & p, int max_new);
long linear_wgs(const LinearParams & p);  // of a launch over segments, or over states
void launch_linear_attention(const LinearParams & p, hipStream_t s);

struct SampleParams {
  int type = 0, vocab = 0, rows = 0;
  long row = 0;
  const void * x = nullptr;
  const float * temperature = nullptr;
  const int32_t * top_k = nullptr;
  const float * top_p = nullptr;
  const float * min_p = nullptr;
  const float * u = nullptr;
  int32_t * token = nullptr;
  // how a call is split, from sample_split
  int pieces = 0, parts = 0, per = 0;  // pieces of a row, work-groups over them and pieces of each; 0 parts: one work-group a row
  void * ws = nullptr;
};
// Sets the split of a call; returns the workspace bytes.
size_t sample_split(SampleParams & p);
void launch_sample(const SampleParams & p, hipStream_t s);

struct RaggedParams {
  int type = 0, heads = 0, group = 1, dim = 0;
  int batch = 0, tokens_q = 0, tokens_k = 0, max_q = 0;
  int causal = 0, window = 0, sinks = 0;
  float scale_log2 = 1.0f;
  const void * q = nullptr;
  const void * k = nullptr;
  const void * v = nullptr;
  void * o = nullptr;
  const int32_t * cu_q = nullptr;
  const int32_t * cu_k = nullptr;
  long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0, o_token = 0, o_head = 0;
};
void launch_ragged_attention(const RaggedParams & p, hipStream_t s);

}  // namespace ivh
