// Serving operators on device memory (include/moonshine_hip.h "serving operators"): a paged key / value cache held in 4 bits --
// its plan, writing, reading and the attention over it -- and the selection and state reordering of a beam search.
// Launchers only: arguments are checked by serve_api.cpp (and trusted here); every launch goes to the given stream, nothing is
// allocated, copied or waited for, so all of them may be captured into a graph.
#pragma once

#include "beam_list.h"
#include "msh_common.h"

namespace msh {

enum class Elem : int { f32 = 0, bf16 = 1, f16 = 2 };
inline size_t elem_bytes(Elem t) { return t == Elem::f32 ? 4 : 2; }

// ---- the cache's form -------------------------------------------------------------------------------------------------
// The unit is a block: 32 tokens of one key / value head, m = ceil(head_dim / 32) groups of 32 elements.  Every (token, group)
// has one power of two 2^(byte - 127) and 32 codes of 4 bits (sign, and an index into 0, .5, 1, 1.5, 2, 3, 4, 6).  A byte holds
// two neighbouring elements of ONE token (the lower in the low nibble), so a token is written without reading what other
// tokens' bytes hold, by any thread, in any order.  Within a block the bytes lie in the order in which the lanes of a wave feed
// them to the matrix instruction (16x16x32: lane = 16 * quarter + index):
//   keys    512 m   [tile 2][up to 4 groups at a time][quarter 4][token 16][group][4]  byte c: elements 32 group + 8 quarter + 2 c, + 1
//   scales   32 m   [token 32][group]
//   values  512 m   [up to 2 groups at a time][quarter 4][pair 16][group][half 2][4]   byte (half, c): token 16 half + 4 quarter + c,
//                                                                                     elements 32 group + 2 pair, + 1
//   scales   32 m   [quarter 4][group][half 2][4]
// A lane's share of a block is 4 m (keys, per tile) and 8 m (values) contiguous bytes.  A page is page_size / 32 blocks of one head,
// the cache [pages][heads][page_size / 32][1088 m].
constexpr int kKv4Block = 32;
__host__ __device__ inline int kv4_groups(int head_dim) { return (head_dim + 31) / 32; }
__host__ __device__ inline int kv4_block_bytes(int m) { return 1088 * m; }

struct Kv4Cache {
  uint8_t* data;
  int64_t pages;
  int32_t heads, page_shift /* log2 of page_size */, head_dim;
};

void page_plan(int32_t* table, int batch, int width, const int32_t* kv_lens, const int32_t* new_lens, const int32_t* row_start,
               int64_t rows, const int32_t* free_pages, int64_t n_free, int page_shift, int64_t* slots, int32_t* used, hipStream_t s);

// element strides (row, head, element)
struct Kv4Rows {
  const void* p;
  int64_t row, head, elem;
};
void kv4_write(const Kv4Cache& c, const Kv4Rows& k, const Kv4Rows& v, Elem type, int64_t rows, const int64_t* slots, hipStream_t s);
void kv4_read(const Kv4Cache& c, const int64_t* slots, int64_t rows, void* k, void* v, Elem type, hipStream_t s);

struct Kv4Attention {
  const void* q;
  void* out;
  float* lse;                 // nullable, [rows][heads]
  int64_t q_row, q_head;      // element strides
  int64_t out_row, out_head;
  const int32_t* table;       // [batch][width]
  const int32_t* kv_lens;     // [batch]
  const int32_t* q_start;     // nullable, [batch + 1]
  float* part;                // nsplit > 1: workspace
  Kv4Cache cache;
  int64_t rows;
  int32_t heads, batch, width, max_q, causal, window, nsplit;
  int32_t tiles, vec;         // set by the launcher, as is the scale's sign (the kernel's scale is its magnitude)
  float sign;
  float scale_log2;           // softmax scale * log2(e)
  uint16_t* fm;               // not null: the engine's decode path takes the output as bf16, fragment-major [rows16][heads * head_dim]
                              // (kernels.h fm16), instead of `out`
  bool fixed;                 // the order of a row's sums goes by nothing that its sequence does not bring along (uniform kernels)
};
constexpr int kPartPad = 4;       // a range's row: 32 m floats, maximum, sum, two unused
// waves per SIMD that the attention's registers allow (tiles of 16 rows)
constexpr int kv4_attention_waves(int groups, bool f32) { return groups <= 2 ? 4 : groups <= 4 && !f32 ? 3 : 2; }
// tile of a wave (16 * rt rows) and waves that share it, or the form for chunks of prompts; see kv4_attention.h
struct Kv4Shape {
  int rt, kw;
  bool chunk;
  int rows() const { return 16 * rt * (chunk ? 4 : 1); }   // of a unit of work
};
Kv4Shape kv4_attention_shape(const Kv4Attention& a, Elem type);
// number of key ranges a launch is split into, and the floats of workspace that takes
int kv4_attention_splits(const Kv4Attention& a, Elem type);
size_t kv4_attention_part_floats(const Kv4Attention& a, int nsplit);
// workgroups of 256 threads along the first axis of a launch: a grid has fewer than 2^32 threads there
constexpr int64_t kGroupsMost = ((int64_t)1 << 24) - 1;
inline int64_t kv4_rows_groups(int64_t rows) { return (rows + 31) / 32 * 8; }                       // of a write or read
inline int64_t kv4_join_groups(int64_t rows, int heads) { return (rows * heads + 3) / 4; }          // of the join, a wave per (row, head)
int64_t kv4_attention_groups(const Kv4Attention& a, Elem type);                                     // of the attention, `nsplit` set
void kv4_attention(const Kv4Attention& a, Elem type, hipStream_t s);

struct BeamSelect {
  const void* logits;
  int64_t row;                // element stride between two beams' rows (row of beam k of entry b: (b * beams + k) * row)
  const float* scores;
  const uint8_t* finished;
  float* out_scores;
  int32_t *parents, *tokens;
  uint8_t* out_finished;
  void* work;
  int32_t batch, beams, vocab, eos;
  bool fixed = false;         // as in Kv4Attention
};
size_t beam_select_work_bytes(int batch, int beams, int vocab, bool fixed = false);
void beam_select(const BeamSelect& a, Elem type, hipStream_t s);

// byte strides; segment (o, b, k, i) starts at data + o * outer_stride + (b * beams + k) * beam_stride + i * inner_stride and holds
// n_rows rows of row_bytes
struct BeamState {
  void* data;
  int64_t outer, outer_stride, beam_stride, inner, inner_stride, row_bytes, n_rows;
};
constexpr int kBeamStates = 4;
int64_t beam_reorder_groups(const BeamState* states, int n_states, int batch);   // workgroups of the launch: below 2^24
void beam_reorder(const BeamState* states, int n_states, int batch, int beams, const int32_t* parents, const int32_t* lengths,
                  int length_stride, hipStream_t s);

// The decode loop around them (Engine::decode_beams).  Row r = clip * beams + beam.  tokens [rows][stride], its [0] = BOS; a beam that had
// ended holds -1 from there on.  pos[0] = steps done, pos[1] = clips still decoding, pos[2] = steps done + 1 (rows of the caches).
struct BeamLoop {
  int32_t *tokens, *pos;
  float *scores, *next_scores;
  uint8_t *finished, *next_finished;
  const int32_t *parents, *picked;
  int32_t stride, beams, clips;
};
void beam_begin(const BeamLoop& l, int bos, const float* embed, int D, float* H, hipStream_t s);
// after the selection and the reordering: append, end what is over its budget (max_len of the row's clip), embed the next inputs
void beam_advance(const BeamLoop& l, const ClipMeta* row_clips, const float* embed, int D, float* H, hipStream_t s);

}  // namespace msh
