// C entry points of the serving operators (include/moonshine_hip.h): every argument that the host can see is checked here, before
// anything is launched; what lives on the device (lengths, page numbers, parents) is bounded by the kernels.  No entry allocates,
// copies or waits.
#include "../../include/moonshine_hip.h"

#include <stdio.h>

#include <algorithm>
#include <string>
#include <utility>

#include "serve_kernels.h"

namespace {

thread_local std::string g_op_error;

template <class F>
int32_t op_guarded(F&& f) {
  try {
    f();
    return MSH_OK;
  } catch (const std::invalid_argument& ex) {
    g_op_error = ex.what();
    return MSH_ERR_INVALID_ARGUMENT;
  } catch (const msh::HipError& ex) {
    g_op_error = ex.what();
    return MSH_ERR_HIP;
  } catch (const std::exception& ex) {
    g_op_error = ex.what();
    return MSH_ERR_UNKNOWN;
  } catch (...) {
    g_op_error = "unknown error";
    return MSH_ERR_UNKNOWN;
  }
}

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

// launches on `device` whatever device the calling thread has current
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(int device) {
    MSH_HIP(hipGetDevice(&before));
    if (before == device) before = -1;
    else MSH_HIP(hipSetDevice(device));
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

constexpr int64_t kMost = (int64_t)1 << 30;   // tokens of a sequence, rows of a call, workgroups of a launch

msh::Elem elem(int32_t dtype) {
  need(dtype == MSH_F32 || dtype == MSH_BF16 || dtype == MSH_F16, "dtype: MSH_F32, MSH_BF16 or MSH_F16");
  return (msh::Elem)dtype;
}

int page_shift(int32_t page_size) {
  need(page_size >= 32 && page_size <= 65536 && (page_size & (page_size - 1)) == 0, "page_size: a power of two from 32 to 65536");
  return __builtin_ctz((unsigned)page_size);
}

msh::Kv4Cache cache_of(const msh_kv4_cache* c) {
  need(c != nullptr, "cache: null");
  need(c->heads >= 1 && c->heads <= 1024, "cache: 1 to 1024 heads");
  need(c->head_dim >= 1 && c->head_dim <= 256, "cache: head_dim from 1 to 256");
  need(c->pages >= 1 && c->pages <= kMost, "cache: 1 to 2^30 pages");
  need(c->data != nullptr && (uintptr_t)c->data % 16 == 0, "cache: data must be a 16-byte aligned device pointer");
  return msh::Kv4Cache{(uint8_t*)c->data, c->pages, c->heads, page_shift(c->page_size), c->head_dim};
}

msh::Kv4Attention attention_of(const msh_kv4_attention_args* x, msh::Elem* type) {
  need(x != nullptr, "args: null");
  msh::Kv4Attention a{};
  *type = elem(x->dtype);
  a.cache = cache_of(&x->cache);
  need(x->heads >= 1 && x->heads <= 65536 && x->heads % a.cache.heads == 0, "heads must be a multiple of the cache's heads");
  need(x->rows >= 0 && x->rows <= kMost && x->batch >= 0 && x->batch <= kMost, "rows and batch: 0 to 2^30");
  need(x->max_q >= 1 && x->max_q <= (1 << 24), "max_q: 1 to 2^24");
  need(x->q_start != nullptr || x->rows == (int64_t)x->batch * x->max_q, "without q_start, rows must be batch * max_q");
  need(x->table_width >= 1 && ((int64_t)x->table_width << a.cache.page_shift) <= kMost, "table_width * page_size: 1 page to 2^30 tokens");
  need(x->causal != 0 || x->window == 0, "window needs causal");
  need(x->window >= 0, "window: 0 (none) or the number of tokens a row sees, its own included");
  need(x->scale == x->scale && x->scale - x->scale == 0.f, "scale must be finite");
  const int64_t per = x->heads / a.cache.heads;
  need((int64_t)x->max_q * per <= kMost, "max_q * heads per cache head: at most 2^30");
  const int64_t tiles = ((int64_t)x->max_q * per + 15) / 16;
  need((double)x->batch * a.cache.heads * tiles < (1 << 24) && x->rows * x->heads < ((int64_t)1 << 32), "the call is too large for one launch");
  a.q = x->q, a.out = x->out, a.lse = x->lse;
  a.q_row = x->q_row_stride, a.q_head = x->q_head_stride, a.out_row = x->out_row_stride, a.out_head = x->out_head_stride;
  a.table = x->block_table, a.kv_lens = x->kv_lens, a.q_start = x->q_start;
  a.rows = x->rows, a.heads = x->heads, a.batch = x->batch, a.width = x->table_width, a.max_q = x->max_q;
  a.causal = x->causal != 0, a.window = x->window;
  a.scale_log2 = x->scale * 1.44269504088896341f;
  a.nsplit = 1;
  if (x->rows > 0 && x->batch > 0) {
    a.nsplit = msh::kv4_attention_splits(a, *type);
    need(msh::kv4_attention_groups(a, *type) <= msh::kGroupsMost, "the call is too large for one launch");
  }
  return a;
}

}  // namespace

extern "C" {

const char* msh_op_last_error(void) { return g_op_error.c_str(); }

int64_t msh_kv4_page_bytes(int32_t heads, int32_t page_size, int32_t head_dim) {
  int64_t n = 0;
  const int32_t rc = op_guarded([&] {
    need(heads >= 1 && heads <= 1024, "heads: 1 to 1024");
    need(head_dim >= 1 && head_dim <= 256, "head_dim: 1 to 256");
    n = (int64_t)heads * ((1 << page_shift(page_size)) / 32) * msh::kv4_block_bytes(msh::kv4_groups(head_dim));
  });
  return rc == MSH_OK ? n : rc;
}

int32_t msh_page_plan(int32_t device, void* stream, int32_t* block_table, int32_t batch, int32_t table_width, const int32_t* kv_lens,
                      const int32_t* new_lens, const int32_t* row_start, int64_t rows, const int32_t* free_pages, int64_t n_free,
                      int32_t page_size, int64_t* slots, int32_t* used) {
  return op_guarded([&] {
    const int shift = page_shift(page_size);
    need(batch >= 1 && batch <= (1 << 20), "batch: 1 to 2^20");
    need(table_width >= 1 && ((int64_t)table_width << shift) <= kMost, "table_width * page_size: 1 page to 2^30 tokens");
    need(rows >= 0 && rows <= kMost, "rows: 0 to 2^30");
    need(n_free >= 0 && n_free <= kMost, "n_free: 0 to 2^30");
    need(block_table && kv_lens && new_lens && row_start && used && (free_pages || n_free == 0) && (slots || rows == 0), "null pointer");
    DeviceScope scope(device);
    msh::page_plan(block_table, batch, table_width, kv_lens, new_lens, row_start, rows, free_pages, n_free, shift, slots, used,
                   (hipStream_t)stream);
  });
}

int32_t msh_kv4_write(int32_t device, void* stream, const msh_kv4_cache* cache, const void* k, const int64_t* k_strides, const void* v,
                      const int64_t* v_strides, int32_t dtype, int64_t rows, const int64_t* slots) {
  return op_guarded([&] {
    const msh::Kv4Cache c = cache_of(cache);
    const msh::Elem t = elem(dtype);
    need(rows >= 0 && rows <= kMost && msh::kv4_rows_groups(rows) <= msh::kGroupsMost, "rows: 0 to 2^26 - 32");
    if (rows == 0) return;
    need(k && v && k_strides && v_strides && slots, "null pointer");
    DeviceScope scope(device);
    msh::kv4_write(c, msh::Kv4Rows{k, k_strides[0], k_strides[1], k_strides[2]}, msh::Kv4Rows{v, v_strides[0], v_strides[1], v_strides[2]}, t,
                   rows, slots, (hipStream_t)stream);
  });
}

int32_t msh_kv4_read(int32_t device, void* stream, const msh_kv4_cache* cache, const int64_t* slots, int64_t rows, void* k, void* v,
                     int32_t dtype) {
  return op_guarded([&] {
    const msh::Kv4Cache c = cache_of(cache);
    const msh::Elem t = elem(dtype);
    need(rows >= 0 && rows <= kMost && msh::kv4_rows_groups(rows) <= msh::kGroupsMost, "rows: 0 to 2^26 - 32");
    if (rows == 0) return;
    need(k && v && slots, "null pointer");
    DeviceScope scope(device);
    msh::kv4_read(c, slots, rows, k, v, t, (hipStream_t)stream);
  });
}

int64_t msh_kv4_attention_workspace(const msh_kv4_attention_args* args) {
  int64_t n = 0;
  const int32_t rc = op_guarded([&] {
    msh::Elem t;
    const msh::Kv4Attention a = attention_of(args, &t);
    n = (int64_t)(msh::kv4_attention_part_floats(a, a.nsplit) * sizeof(float));
  });
  return rc == MSH_OK ? n : rc;
}

int32_t msh_kv4_attention(int32_t device, void* stream, const msh_kv4_attention_args* args, void* workspace, int64_t workspace_bytes) {
  return op_guarded([&] {
    msh::Elem t;
    msh::Kv4Attention a = attention_of(args, &t);
    if (a.rows == 0 || a.batch == 0) return;
    need(a.q && a.out && a.table && a.kv_lens, "null pointer");
    const int64_t want = (int64_t)(msh::kv4_attention_part_floats(a, a.nsplit) * sizeof(float));
    need(want == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= want),
         "workspace: smaller than msh_kv4_attention_workspace() says, or not 16-byte aligned");
    a.part = (float*)workspace;
    DeviceScope scope(device);
    msh::kv4_attention(a, t, (hipStream_t)stream);
  });
}

static void select_sizes(int32_t batch, int32_t beams, int32_t vocab) {
  need(batch >= 0 && batch <= (1 << 21), "batch: 0 to 2^21");
  need(beams >= 1 && beams <= msh::kBeamMax, "beams: 1 to 16");
  need(vocab >= 1 && vocab <= (1 << 24), "vocab: 1 to 2^24");
}

int64_t msh_beam_select_workspace(int32_t batch, int32_t beams, int32_t vocab) {
  int64_t n = 0;
  const int32_t rc = op_guarded([&] {
    select_sizes(batch, beams, vocab);
    n = batch == 0 ? 0 : (int64_t)msh::beam_select_work_bytes(batch, beams, vocab);
  });
  return rc == MSH_OK ? n : rc;
}

int32_t msh_beam_select(int32_t device, void* stream, const void* logits, int32_t dtype, int64_t row_stride, int32_t batch, int32_t beams,
                        int32_t vocab, const float* scores, const uint8_t* finished, int32_t eos, float* next_scores, int32_t* parents,
                        int32_t* tokens, uint8_t* next_finished, void* workspace, int64_t workspace_bytes) {
  return op_guarded([&] {
    const msh::Elem t = elem(dtype);
    select_sizes(batch, beams, vocab);
    need(eos >= -1 && eos < vocab, "eos: an id of the vocabulary, or -1 for none");
    if (batch == 0) return;
    need(row_stride >= 0, "row_stride: not negative");
    need(logits && scores && finished && next_scores && parents && tokens && next_finished, "null pointer");
    need((uintptr_t)logits % msh::elem_bytes(t) == 0, "logits: not aligned to their type");
    need(next_scores != scores && next_finished != finished, "next_scores and next_finished must not be the inputs");
    need(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= (int64_t)msh::beam_select_work_bytes(batch, beams, vocab),
         "workspace: smaller than msh_beam_select_workspace() says, or not 16-byte aligned");
    DeviceScope scope(device);
    msh::beam_select(msh::BeamSelect{logits, row_stride, scores, finished, next_scores, parents, tokens, next_finished, workspace, batch, beams,
                                     vocab, eos},
                     t, (hipStream_t)stream);
  });
}

// no two of a state's (outer, entry and beam, inner) pieces of `bytes` share a byte: from the smallest stride up, each steps over what lies below
static void apart(const msh_beam_state& x, int64_t bytes, int64_t rows) {
  if (bytes == 0 || x.outer == 0 || x.inner == 0) return;
  std::pair<int64_t, int64_t> by[3] = {{x.outer_stride, x.outer}, {x.beam_stride, rows}, {x.inner_stride, x.inner}};
  std::sort(by, by + 3);
  double extent = (double)bytes;
  for (const auto& d : by) {
    if (d.second == 1) continue;
    need((double)d.first >= extent, "state: its rows overlap");
    extent += (double)d.first * (double)(d.second - 1);
  }
}

int32_t msh_beam_reorder(int32_t device, void* stream, const msh_beam_state* states, int32_t n_states, int32_t batch, int32_t beams,
                         const int32_t* parents, const int32_t* lengths, int32_t length_stride) {
  return op_guarded([&] {
    need(batch >= 0 && batch <= (1 << 24), "batch: 0 to 2^24");
    need(beams >= 1 && beams <= msh::kBeamMax, "beams: 1 to 16");
    need(n_states >= 0 && n_states <= msh::kBeamStates && (states || n_states == 0), "states: 0 to 4");
    need(length_stride == 0 || length_stride == 1, "length_stride: 0 (one length for all) or 1");
    if (batch == 0 || n_states == 0) return;
    need(parents != nullptr, "null pointer");
    msh::BeamState st[msh::kBeamStates];
    for (int i = 0; i < n_states; ++i) {
      const msh_beam_state& x = states[i];
      need(x.outer >= 0 && x.inner >= 0 && x.row_bytes >= 0 && x.n_rows >= 0 && x.outer <= kMost && x.inner <= kMost && x.row_bytes <= kMost &&
               x.n_rows <= kMost, "state: sizes from 0 to 2^30");
      const int64_t bytes = x.row_bytes * x.n_rows;
      need(bytes <= ((int64_t)1 << 40), "state: a beam's rows are too large");
      need(x.outer == 0 || x.inner == 0 || bytes == 0 || x.data != nullptr, "null pointer");
      need((double)x.outer * x.inner * batch * (double)(bytes / 256 + 1) < 2147483648.0, "state: too large for one launch");
      apart(x, bytes, (int64_t)batch * beams);
      for (int j = 0; j < i; ++j) need(x.data != states[j].data || x.data == nullptr, "states: the same address twice");
      st[i] = msh::BeamState{x.data, x.outer, x.outer_stride, x.beam_stride, x.inner, x.inner_stride, x.row_bytes, x.n_rows};
    }
    need(msh::beam_reorder_groups(st, n_states, batch) < (1 << 24), "states: too large for one launch");   // (a grid has 2^32 threads)
    DeviceScope scope(device);
    msh::beam_reorder(st, n_states, batch, beams, parents, lengths, length_stride, (hipStream_t)stream);
  });
}

}  // extern "C"
