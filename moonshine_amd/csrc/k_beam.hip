// Beam search: selection over beams and vocabulary, reordering of the states that the selected beams continue.
#include <float.h>

#include "kernels.h"
#include "kv4_common.h"

namespace msh {
namespace {

__device__ __forceinline__ void wave_fence() {   // shared memory written by one lane of a wave, read by another
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- selection ----------------------------------------------------------------------------------------------------------
// score(k, v) = score_k + l_kv - log sum_v exp l_kv; the `beams` best of all (k, v), ties to the lowest k * vocab + v.
// Pass 1, one wave per (row, part): running maximum and sum of exponentials, and the part's `beams` best logits in order -- the order
//   inside a row does not depend on its sum.  Elements stay in registers (32 a lane): the K-th largest of the 64 lanes' maxima bounds
//   the K-th largest element from below, so that all but a handful are dismissed by one comparison; later elements are held
//   against the K-th best found so far.  One read of the logits: bound by HBM bandwidth for batches, by latency for one clip.
// Pass 2, one workgroup per batch entry: joins the parts, ranks beams * parts * beams candidates.
// The sums are added in 64 bits from 32 exponentials at a time and the scores compared in 64 bits: the order of two candidates of
// different beams hangs on both rows' sums.
struct Part {
  double sum;
  float top;
  int pad;
};
struct Entry {
  float val;
  int idx;
};
__host__ __device__ inline size_t part_bytes(int beams) { return sizeof(Part) + sizeof(Entry) * beams; }

constexpr int kLane = 32;                               // elements of a lane per chunk
constexpr int kListMax = kBeamMax * kLane + 2 * kBeamMax;   // elements above the bound lie in at most K lanes; K earlier ones, K ties

__device__ __forceinline__ bool before(const Entry& a, const Entry& b) { return a.val > b.val || (a.val == b.val && a.idx < b.idx); }

template <Elem E>
__global__ __launch_bounds__(256) void beam_partial_kernel(BeamSelect a, int parts, uint8_t* work) {
  typedef typename ElemOf<E>::T T;
  constexpr int VEC = 16 / sizeof(T), LOADS = kLane / VEC;
  __shared__ Entry list_s[4][kListMax];
  __shared__ Entry best_s[4][kBeamMax];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  const int64_t row = id / parts;
  const int part = (int)(id % parts);
  if (row >= (int64_t)a.batch * a.beams) return;
  const float score = a.scores[row];
  if (a.finished[row] != 0 || !(score > -INFINITY)) return;   // its logits are not looked at
  Entry* list = list_s[wave];
  Entry* best = best_s[wave];
  const int K = a.beams;

  // whole 16-byte vectors from the one that holds the row's first element: each holds an element of the row, so none leaves its memory
  const T* p = static_cast<const T*>(a.logits) + row * a.row;
  const int off = (int)(((uintptr_t)p & 15) / sizeof(T));
  const uint4* vec = reinterpret_cast<const uint4*>(p - off);
  const int nv = (a.vocab + off + VEC - 1) / VEC;
  const int per = ((nv + parts - 1) / parts + 63) & ~63;
  const int v0 = part * per, v1 = v0 + per < nv ? v0 + per : nv;

  float top = -INFINITY;    // of this lane
  double sum = 0.0;
  int have = 0;             // entries of `best`
  for (int base = v0; base < v1; base += 64 * LOADS) {
    float x[kLane];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int i = base + l * 64 + lane;
      const uint4 u = i < v1 ? vec[i] : uint4{0, 0, 0, 0};
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[l * 4 + e] = __uint_as_float(w[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[l * 8 + 2 * e] = ElemOf<E>::get((T)w[e]), x[l * 8 + 2 * e + 1] = ElemOf<E>::get((T)(w[e] >> 16));
      }
    }
    if (base * VEC < off || (base + 64 * LOADS) * VEC > a.vocab + off || base + 64 * LOADS > v1) {
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        const int i = base + (e / VEC) * 64 + lane, idx = i * VEC + e % VEC - off;
        if (i >= v1 || idx < 0 || idx >= a.vocab) x[e] = -INFINITY;
      }
    }
    float hi = -INFINITY, now, part_sum;
    auto sums = [&] {
      hi = -INFINITY;
#pragma unroll
      for (int e = 0; e < kLane; ++e) hi = fmaxf(hi, x[e]);
      now = fmaxf(top, hi);
      const float ref = now == -INFINITY ? 0.f : now;
      part_sum = 0.f;
#pragma unroll
      for (int e = 0; e < kLane; ++e) part_sum += __builtin_amdgcn_exp2f((x[e] - ref) * 1.44269504088896341f);
    };
    sums();
    if (__builtin_amdgcn_ballot_w64(!(part_sum < INFINITY)) != 0) {   // NaN counts as -inf, +inf as the largest finite value
#pragma unroll
      for (int e = 0; e < kLane; ++e) x[e] = x[e] != x[e] ? -INFINITY : fminf(x[e], FLT_MAX);
      sums();
    }
    if (now > top) {
      sum *= top == -INFINITY ? 0.0 : (double)__builtin_amdgcn_exp2f((top - now) * 1.44269504088896341f);
      top = now;
    }
    sum += (double)part_sum;

    // bound: K entries found -> only what is better counts; otherwise the K-th largest lane maximum
    float bound = have == K ? best[K - 1].val : -INFINITY;
    if (__builtin_amdgcn_ballot_w64(hi > bound) == 0) continue;
    bool strict = have == K;   // an equal value has a higher index than what was found before
    if (__popcll(__builtin_amdgcn_ballot_w64(hi > bound)) > K) {
      float left = hi;
      float kth = -INFINITY;
      for (int k = 0; k < K; ++k) {
        kth = left;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) kth = fmaxf(kth, __shfl_xor(kth, o));
        const uint64_t at = __builtin_amdgcn_ballot_w64(left == kth);
        if (lane == __ffsll((unsigned long long)at) - 1) left = -INFINITY;
      }
      if (kth > bound) bound = kth, strict = false;
    }
    int n = 0;
    for (int k = lane; k < have; k += 64) list[k] = best[k];
    n = have;
    if (__builtin_amdgcn_ballot_w64(hi > bound) != 0) {
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        const bool in = x[e] > bound;
        const uint64_t m = __builtin_amdgcn_ballot_w64(in);
        if (m != 0) {
          const int at = n + __popcll(m & ((1ull << lane) - 1));
          if (in) list[at] = Entry{x[e], (base + (e / VEC) * 64 + lane) * VEC + e % VEC - off};
          n += __popcll(m);
        }
      }
    }
    // equal to the bound: the lowest indices, as many as can still count
    if (!strict && bound > -INFINITY) {
      int next = INT_MAX;   // this lane's lowest index not taken yet
      auto seek = [&](int after) {
        next = INT_MAX;
#pragma unroll
        for (int e = kLane - 1; e >= 0; --e) {
          const int idx = (base + (e / VEC) * 64 + lane) * VEC + e % VEC - off;
          if (x[e] == bound && idx > after) next = idx;
        }
      };
      seek(-1);
      for (int k = n - have; k < K; ++k) {
        int lowest = next;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) lowest = min(lowest, __shfl_xor(lowest, o));
        if (lowest == INT_MAX) break;
        if (next == lowest) {
          list[n] = Entry{bound, lowest};
          seek(lowest);
        }
        ++n;
      }
    }
    wave_fence();
    // rank by counting
    const int keep = n < K ? n : K;
    for (int i = lane; i < n; i += 64) {
      const Entry mine = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += before(list[j], mine) ? 1 : 0;
      if (rank < K) best[rank] = mine;
    }
    have = keep;
    wave_fence();
  }

  float all = top;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  double total = top == -INFINITY ? 0.0 : sum * exp((double)top - (double)all);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o);
  uint8_t* out = work + (row * parts + part) * part_bytes(K);
  if (lane == 0) *reinterpret_cast<Part*>(out) = Part{total, all, 0};
  if (lane < K) reinterpret_cast<Entry*>(out + sizeof(Part))[lane] = lane < have ? best[lane] : Entry{-INFINITY, INT_MAX};
}

constexpr int kCandidates = 16;   // of a thread of pass 2

__global__ __launch_bounds__(256) void beam_pick_kernel(BeamSelect a, int parts, const uint8_t* work) {
  __shared__ double offset_s[kBeamMax];
  __shared__ double top_s[4];
  __shared__ int64_t flat_s[4];
  __shared__ double picked_s[kBeamMax];
  __shared__ int64_t picked_flat_s[kBeamMax];
  const int K = a.beams, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * K;
  if (threadIdx.x < K) {   // score_k - log sum exp of row k; NaN: a finished or dead beam
    const int64_t row = row0 + threadIdx.x;
    double o = __builtin_nan("");
    if (a.finished[row] == 0 && a.scores[row] > -INFINITY) {
      float top = -INFINITY;
      for (int p = 0; p < parts; ++p) top = fmaxf(top, reinterpret_cast<const Part*>(work + (row * parts + p) * part_bytes(K))->top);
      double sum = 0.0;
      for (int p = 0; p < parts; ++p) {
        const Part* q = reinterpret_cast<const Part*>(work + (row * parts + p) * part_bytes(K));
        if (q->top > -INFINITY) sum += q->sum * exp((double)q->top - (double)top);
      }
      if (top > -INFINITY) o = (double)a.scores[row] - (log(sum) + (double)top);
    }
    offset_s[threadIdx.x] = o;
  }
  __syncthreads();
  double val[kCandidates];
  int64_t flat[kCandidates];
  const int total = K * parts * K;
#pragma unroll
  for (int c = 0; c < kCandidates; ++c) {
    val[c] = -INFINITY, flat[c] = INT64_MAX;
    const int i = c * 256 + (int)threadIdx.x;
    if (i >= total) continue;
    const int k = i / (parts * K), p = i / K % parts, e = i % K;
    const int64_t row = row0 + k;
    if (a.finished[row] != 0) {
      if (p == 0 && e == 0 && a.scores[row] > -INFINITY) val[c] = a.scores[row], flat[c] = (int64_t)k * a.vocab + (a.eos > 0 ? a.eos : 0);
      continue;
    }
    const double o = offset_s[k];
    if (!(o == o)) continue;
    const Entry en = reinterpret_cast<const Entry*>(work + (row * parts + p) * part_bytes(K) + sizeof(Part))[e];
    if (en.val > -INFINITY) val[c] = o + (double)en.val, flat[c] = (int64_t)k * a.vocab + en.idx;
  }
  for (int k = 0; k < K; ++k) {
    double v = -INFINITY;
    int64_t f = INT64_MAX;
#pragma unroll
    for (int c = 0; c < kCandidates; ++c)
      if (val[c] > v || (val[c] == v && flat[c] < f)) v = val[c], f = flat[c];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const double v2 = __shfl_xor(v, o);
      const int64_t f2 = __shfl_xor(f, o);
      if (v2 > v || (v2 == v && f2 < f)) v = v2, f = f2;
    }
    if (lane == 0) top_s[wave] = v, flat_s[wave] = f;
    __syncthreads();
    v = top_s[0], f = flat_s[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
      if (top_s[w] > v || (top_s[w] == v && flat_s[w] < f)) v = top_s[w], f = flat_s[w];
#pragma unroll
    for (int c = 0; c < kCandidates; ++c)
      if (flat[c] == f) val[c] = -INFINITY, flat[c] = INT64_MAX;
    if (threadIdx.x == 0) picked_s[k] = v, picked_flat_s[k] = f;
    __syncthreads();
  }
  if (threadIdx.x < K) {
    const int k = threadIdx.x;
    const int64_t row = row0 + k, f = picked_flat_s[k];
    const bool empty = f == INT64_MAX;
    const int parent = empty ? k : (int)(f / a.vocab), token = empty || a.finished[row0 + parent] != 0 ? a.eos : (int)(f % a.vocab);
    const uint8_t done = empty || a.finished[row0 + parent] != 0 || token == a.eos;
    a.out_scores[row] = (float)picked_s[k];
    a.parents[row] = parent;
    a.tokens[row] = token;
    a.out_finished[row] = done;
  }
}

int beam_parts(int batch, int beams, int vocab) {
  const int64_t rows = (int64_t)batch * beams;
  int64_t n = (8192 + rows - 1) / rows;                         // waves that fill the chip
  const int64_t chunks = (vocab + 64 * kLane - 1) / (64 * kLane);
  n = n < chunks ? n : chunks;
  const int64_t most = 256 * kCandidates / ((int64_t)beams * beams);
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n);
}

// ---- reordering ---------------------------------------------------------------------------------------------------------
// state[b, k, :len_b] <- state[b, parent[b, k], :len_b] in place.  A thread owns one piece (16 bytes) of all beams of (outer, b, inner): it
// loads what its beams' parents have there, then stores -- no thread reads what another writes, whatever the parents are, and a beam
// that continues itself is neither read nor written.  Bound by HBM bandwidth.
struct BeamStates {
  BeamState s[kBeamStates];
  int64_t first[kBeamStates + 1];   // first workgroup of each state
  int32_t blocks[kBeamStates];      // workgroups of one (outer, b, inner)
  int32_t unit[kBeamStates];        // bytes of a piece: 16, 4 or 1, as the state's address and strides allow
};

template <int KMAX, class P>
__device__ __forceinline__ void move_piece(uint8_t* p, int64_t stride, const int32_t* parents, int beams, int bytes) {
  P v[KMAX];
#pragma unroll
  for (int k = 0; k < KMAX; ++k) {
    const int from = k < beams ? parents[k] : k;
    if (from != k && from >= 0 && from < beams) v[k] = *reinterpret_cast<const P*>(p + from * stride);
  }
#pragma unroll
  for (int k = 0; k < KMAX; ++k) {
    const int from = k < beams ? parents[k] : k;
    if (from == k || from < 0 || from >= beams) continue;
    if (bytes >= (int)sizeof(P)) {
      *reinterpret_cast<P*>(p + k * stride) = v[k];
    } else {   // the last piece of the valid rows
      const uint8_t* w = reinterpret_cast<const uint8_t*>(&v[k]);
#pragma unroll
      for (int i = 0; i < (int)sizeof(P); ++i)
        if (i < bytes) p[k * stride + i] = w[i];
    }
  }
}

template <int KMAX>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamStates all, int n_states, int batch, int beams, const int32_t* parents,
                                                           const int32_t* lengths, int length_stride) {
  const int64_t block = blockIdx.x;
  int which = 0;
  while (which + 1 < n_states && block >= all.first[which + 1]) ++which;
  const BeamState& s = all.s[which];
  const int64_t at = block - all.first[which], seg = at / all.blocks[which];
  const int64_t inner = seg % s.inner, b = seg / s.inner % batch, outer = seg / s.inner / batch;
  int64_t rows = lengths != nullptr ? lengths[b * length_stride] : s.n_rows;
  rows = rows < 0 ? 0 : rows > s.n_rows ? s.n_rows : rows;
  const int64_t bytes = rows * s.row_bytes;
  uint8_t* p = static_cast<uint8_t*>(s.data) + outer * s.outer_stride + b * beams * s.beam_stride + inner * s.inner_stride;
  const int32_t* par = parents + b * beams;
  const int64_t piece = (at % all.blocks[which]) * 256 + threadIdx.x;
  const int64_t o = piece * all.unit[which];
  if (o >= bytes) return;
  if (all.unit[which] == 16) move_piece<KMAX, uint4>(p + o, s.beam_stride, par, beams, (int)(bytes - o < 16 ? bytes - o : 16));
  else if (all.unit[which] == 4) move_piece<KMAX, uint32_t>(p + o, s.beam_stride, par, beams, (int)(bytes - o < 4 ? bytes - o : 4));
  else move_piece<KMAX, uint8_t>(p + o, s.beam_stride, par, beams, 1);
}

// ---- the decode loop ----------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(128) void beam_begin_kernel(BeamLoop l, int bos, const float* __restrict__ embed, int D, float* __restrict__ H) {
  const int row = blockIdx.x;
  if (threadIdx.x == 0) {
    l.tokens[(int64_t)row * l.stride] = bos;
    l.scores[row] = row % l.beams == 0 ? 0.f : -INFINITY;   // all beams grow from one
    l.finished[row] = 0;
    if (row == 0) l.pos[0] = 0, l.pos[1] = l.clips, l.pos[2] = 1;
  }
  for (int d = threadIdx.x; d < D; d += 128) H[fm32(row, d, D >> 5)] = embed[(int64_t)bos * D + d];
}

// one workgroup per clip: its beams' old flags are read before any is written
__global__ __launch_bounds__(256) void beam_advance_kernel(BeamLoop l, const ClipMeta* __restrict__ row_clips, const float* __restrict__ embed,
                                                           int D, float* __restrict__ H) {
  __shared__ uint8_t was_s[kBeamMax], now_s[kBeamMax];
  const int row0 = blockIdx.x * l.beams, k = threadIdx.x, pos = l.pos[0];
  if (k < l.beams) was_s[k] = l.finished[row0 + k];
  __syncthreads();
  if (k < l.beams) {
    const int row = row0 + k;
    const bool over = was_s[l.parents[row]] != 0;
    l.tokens[(int64_t)row * l.stride + pos + 1] = over ? -1 : l.picked[row];
    now_s[k] = l.next_finished[row] != 0 || pos + 1 >= row_clips[row].max_len;
    l.finished[row] = now_s[k];
    l.scores[row] = l.next_scores[row];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    bool was = true, now = true;
    for (int i = 0; i < l.beams; ++i) was = was && was_s[i] != 0, now = now && now_s[i] != 0;
    if (now && !was) atomicSub(l.pos + 1, 1);
  }
  for (int i = threadIdx.x; i < l.beams * D; i += 256) {
    const int row = row0 + i / D, d = i % D;
    const int id = l.picked[row];
    H[fm32(row, d, D >> 5)] = embed[(int64_t)(id < 0 ? 0 : id) * D + d];
  }
}

__global__ void beam_tick_kernel(int32_t* pos) {
  pos[0] += 1;
  pos[2] += 1;
}

}  // namespace

void beam_begin(const BeamLoop& l, int bos, const float* embed, int D, float* H, hipStream_t s) {
  MSH_LAUNCH(beam_begin_kernel, dim3(l.clips * l.beams), dim3(128), 0, s, l, bos, embed, D, H);
}
void beam_advance(const BeamLoop& l, const ClipMeta* row_clips, const float* embed, int D, float* H, hipStream_t s) {
  MSH_LAUNCH(beam_advance_kernel, dim3(l.clips), dim3(256), 0, s, l, row_clips, embed, D, H);
  MSH_LAUNCH(beam_tick_kernel, dim3(1), dim3(1), 0, s, l.pos);
}

size_t beam_select_work_bytes(int batch, int beams, int vocab) {
  return (size_t)batch * beams * beam_parts(batch, beams, vocab) * part_bytes(beams);
}

void beam_select(const BeamSelect& a, Elem type, hipStream_t s) {
  const int parts = beam_parts(a.batch, a.beams, a.vocab);
  const dim3 grid((unsigned)(((int64_t)a.batch * a.beams * parts + 3) / 4));
  uint8_t* work = static_cast<uint8_t*>(a.work);
  if (type == Elem::f32) MSH_LAUNCH((beam_partial_kernel<Elem::f32>), grid, dim3(256), 0, s, a, parts, work);
  else if (type == Elem::bf16) MSH_LAUNCH((beam_partial_kernel<Elem::bf16>), grid, dim3(256), 0, s, a, parts, work);
  else MSH_LAUNCH((beam_partial_kernel<Elem::f16>), grid, dim3(256), 0, s, a, parts, work);
  MSH_LAUNCH(beam_pick_kernel, dim3(a.batch), dim3(256), 0, s, a, parts, work);
}

void beam_reorder(const BeamState* states, int n_states, int batch, int beams, const int32_t* parents, const int32_t* lengths,
                  int length_stride, hipStream_t s) {
  BeamStates all{};
  int64_t blocks = 0;
  int n = 0;
  for (int i = 0; i < n_states; ++i) {
    const BeamState& st = states[i];
    const int64_t bytes = st.n_rows * st.row_bytes;
    if (bytes == 0 || st.outer == 0 || st.inner == 0) continue;
    all.s[n] = st;
    all.first[n] = blocks;
    auto fits = [&](int64_t u) {
      return (uintptr_t)st.data % u == 0 && (st.outer == 1 || st.outer_stride % u == 0) && st.beam_stride % u == 0 &&
             (st.inner == 1 || st.inner_stride % u == 0);
    };
    all.unit[n] = fits(16) ? 16 : fits(4) ? 4 : 1;
    all.blocks[n] = (int32_t)((bytes + 256 * all.unit[n] - 1) / (256 * all.unit[n]));
    blocks += st.outer * batch * st.inner * all.blocks[n];
    ++n;
  }
  if (n == 0 || beams < 2) return;
  all.first[n] = blocks;
  if (beams <= 4) MSH_LAUNCH(beam_reorder_kernel<4>, dim3((unsigned)blocks), dim3(256), 0, s, all, n, batch, beams, parents, lengths, length_stride);
  else if (beams <= 8) MSH_LAUNCH(beam_reorder_kernel<8>, dim3((unsigned)blocks), dim3(256), 0, s, all, n, batch, beams, parents, lengths, length_stride);
  else MSH_LAUNCH(beam_reorder_kernel<16>, dim3((unsigned)blocks), dim3(256), 0, s, all, n, batch, beams, parents, lengths, length_stride);
}

}  // namespace msh
