// Host side of the sequence operators: rotary positions, paged key/value cache, attention over
// it and over ragged rows.  Parameter blocks are fully checked by the C ABI (seq_api.cpp)
// before a launch; what only the device knows (lengths, page numbers) the kernels check.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace ivh {

enum SeqType : int { kSeqF16 = 0, kSeqBF16 = 1 };

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
};
// Sets the split of a call with at most max_new new tokens and max_len cached ones in a
// sequence (bounds that only steer the split); returns the workspace bytes.
size_t paged_split(PagedParams & p, int max_new, int max_len);
void launch_paged_attention(const PagedParams & p, hipStream_t s);
void launch_paged_bf16(const PagedParams & p, hipStream_t s);  // its bf16 kernels, built by themselves

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
