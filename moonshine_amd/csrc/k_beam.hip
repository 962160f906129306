// Beam search: selection over beams and vocabulary, reordering of the states that the selected beams continue.
#include <float.h>

#include "beam_list.h"
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
//   inside a row does not depend on its sum.  Elements stay in registers (32 a lane); the next 32 are in flight.  The K-th largest of
//   the 64 lanes' maxima bounds the K-th largest element from below, so that all but a handful are dismissed by one comparison;
//   later elements are held against that bound, which rises again where what passes could fill the list (beam_list.h), and the list of what passed is
//   ranked once.  One read of the logits.  Bound by the vector unit for batches (61 % busy: 19 instructions for 64 logits, fixed work of each part among
//   them), by latency (and the fetch of its own instructions: rare paths are loops, not copies) for one clip.
// Pass 2, one workgroup per batch entry, a thread per (row, part): joins the rows' sums, takes from the parts' lists what reaches the K-th
//   largest list head of a wave, ranks those few by counting.  Bound by the latency of its chain of steps.
// 256 entries of 8 beams over 32768 bf16 logits (a sixth of the beams finished: 114 MB): 41 us, 2.8 TB/s, and 9.6 us; 1 entry of 4 beams, 32-bit logits:
// 6.6 and 4.0 us; 1 entry of 7 beams over 193263 (bf16): 10.4 and 6.2 us; 17 of 10 over 86111: 19.3 and 8.2 us.  Logits that rise all along a row, so that
// every chunk passes the bound of the one before, are the dearest: the first of these takes 133 us a call instead of 53.
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
__host__ __device__ inline size_t part_bytes(int beams) { return sizeof(Part) + sizeof(Entry) * ((beams + 1) & ~1); }   // (16-byte multiples)

constexpr int kPartsMax = 64;                                  // a row's parts lie in one wave of pass 2

__device__ __forceinline__ bool before(const Entry& a, const Entry& b) { return a.val > b.val || (a.val == b.val && a.idx < b.idx); }

// reductions over the wave along the lanes' own paths (row shifts, row broadcasts): no shared memory; the result in every lane
template <int CTRL>
__device__ __forceinline__ float lanes_max(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = lanes_max<0x111>(v);   // row_shr 1, 2, 4, 8, row_bcast 15, 31
  v = lanes_max<0x112>(v);
  v = lanes_max<0x114>(v);
  v = lanes_max<0x118>(v);
  v = lanes_max<0x142>(v);
  v = lanes_max<0x143>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// the K-th largest of the lanes' values, one lane taken away each time
__device__ __forceinline__ float wave_kth(float v, int K, int lane) {
  float kth = -INFINITY;
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    kth = wave_max(v);
    const uint64_t at = __builtin_amdgcn_ballot_w64(v == kth);
    if (lane == __ffsll((unsigned long long)at) - 1) v = -INFINITY;
  }
  return kth;
}

// list[0 .. n) -> the K best in order, by counting; returns how many there are
__device__ __forceinline__ int rank_list(const Entry* list, Entry* best, int n, int K, int lane) {
  wave_fence();
#pragma unroll 1
  for (int i = lane; i < n; i += 64) {
    const Entry mine = list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += before(list[j], mine) ? 1 : 0;
    if (rank < K) best[rank] = mine;
  }
  wave_fence();
  return n < K ? n : K;
}

// (waves per SIMD: at five the 32-bit form spills)
template <Elem E>
__global__ __launch_bounds__(256, (E == Elem::f32 ? 4 : 5)) void beam_partial_kernel(BeamSelect a, int parts, uint8_t* work) {
  typedef typename ElemOf<E>::T T;
  constexpr int VEC = 16 / sizeof(T), LOADS = kLane / VEC;
  __shared__ Entry list_s[4][kListMax];
  __shared__ Entry best_s[4][kBeamMax];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = (int)blockIdx.x * 4 + wave, row = id / parts, part = id - row * parts;
  if (row >= a.batch * a.beams) return;
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
  int n = 0;                // entries of the list
  float bound = -INFINITY;  // every element that can be among the K best so far and is not in the list yet is above it
  bool enough = false;      // K elements of the list reach the bound
  uint4 raw[LOADS];
  auto fetch = [&](int base) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int i = base + l * 64 + lane;
      raw[l] = i < v1 ? vec[i] : uint4{0, 0, 0, 0};
    }
  };
  fetch(v0);
#pragma unroll 1
  for (int base = v0; base < v1; base += 64 * LOADS) {
    float x[kLane];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const uint32_t w[4] = {raw[l].x, raw[l].y, raw[l].z, raw[l].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) x[l * 4 + e] = __uint_as_float(w[e]);
        else if constexpr (E == Elem::bf16) x[l * 8 + 2 * e] = __uint_as_float(w[e] << 16), x[l * 8 + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        else x[l * 8 + 2 * e] = ElemOf<E>::get((T)w[e]), x[l * 8 + 2 * e + 1] = ElemOf<E>::get((T)(w[e] >> 16));
      }
    }
    if (base + 64 * LOADS < v1) fetch(base + 64 * LOADS);
    // index of this lane's element 0; element e: + (e / VEC) * 64 * VEC + e % VEC.  (Copies that the compiler takes for different:
    // otherwise it computes 32 indices once and keeps them in as many registers.)
    const int first = base * VEC + lane * VEC - off;
    int first_push = first, first_tie = first;
    asm("" : "+v"(first_push));
    asm("" : "+v"(first_tie));
    if (base == 0 || base + 64 * LOADS >= v1) {        // the row's ends and the part's: places [lo, lo + span) of the chunk count
      asm volatile("" ::: );
      const int lo = base == 0 ? off : 0, end = min(v1 * VEC, a.vocab + off) - base * VEC;
      const uint32_t span = (uint32_t)(end - lo);
      uint32_t at = (uint32_t)(lane * VEC - lo);
#pragma unroll
      for (int e = 0; e < kLane; ++e)
        if (at + (uint32_t)((e / VEC) * 64 * VEC + e % VEC) >= span) x[e] = -INFINITY;
    }
    float hi, group[4], now, part_sum;
    while (true) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        group[q] = x[8 * q];
#pragma unroll
        for (int e = 1; e < 8; ++e) group[q] = fmaxf(group[q], x[8 * q + e]);
      }
      hi = fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3]));
      now = fmaxf(top, hi);
      const float ref = now == -INFINITY ? 0.f : now;
      part_sum = 0.f;
#pragma unroll
      for (int e = 0; e < kLane; ++e) part_sum += __builtin_amdgcn_exp2f((x[e] - ref) * 1.44269504088896341f);
      if (__builtin_amdgcn_ballot_w64(!(part_sum < INFINITY)) == 0) break;
      // NaN counts as -inf, +inf as the largest finite value
#pragma unroll
      for (int e = 0; e < kLane; ++e) x[e] = x[e] != x[e] ? -INFINITY : fminf(x[e], FLT_MAX);
    }
    if (now > top) {
      sum *= top == -INFINITY ? 0.0 : (double)__builtin_amdgcn_exp2f((top - now) * 1.44269504088896341f);
      top = now;
    }
    sum += (double)part_sum;

    // what is above the bound joins the list; where the list's room asks for it (beam_list.h), the K-th largest lane maximum becomes the bound
    int over = __popcll(__builtin_amdgcn_ballot_w64(hi > bound));
    if (over == 0) continue;
    if (beam_list_cut(n, K)) {
      n = rank_list(list, best, n, K, lane);
      if (lane < n) list[lane] = best[lane];
      if (n == K) bound = fmaxf(bound, best[K - 1].val), enough = true;
      wave_fence();
      over = __popcll(__builtin_amdgcn_ballot_w64(hi > bound));
    }
    const bool raise = beam_bound_rises(n, K, over, enough);   // (more than K lanes are above the bound: it rises)
    if (raise) bound = wave_kth(hi, K, lane);
    const int n0 = n;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (__builtin_amdgcn_ballot_w64(group[q] > bound) == 0) continue;
#pragma unroll
      for (int e = 8 * q; e < 8 * q + 8; ++e) {
        const bool in = x[e] > bound;
        const uint64_t m = __builtin_amdgcn_ballot_w64(in);
        if (m != 0) {
          if (in) list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = Entry{x[e], first_push + (e / VEC) * 64 * VEC + e % VEC};
          n += __popcll(m);
        }
      }
    }
    if (raise) {   // equal to the bound: the lowest indices, as many as can still count (in later chunks an equal value comes behind them)
      int after = -1;
#pragma unroll 1
      for (int k = n - n0; k < K; ++k) {
        int next = INT_MAX;   // this lane's lowest index behind `after`
#pragma unroll
        for (int e = kLane - 1; e >= 0; --e) {
          const int idx = first_tie + (e / VEC) * 64 * VEC + e % VEC;
          if (x[e] == bound && idx > after) next = idx;
        }
        int lowest = next;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) lowest = min(lowest, __shfl_xor(lowest, o));
        if (lowest == INT_MAX) break;
        if (next == lowest) list[n] = Entry{bound, lowest};
        after = lowest;
        ++n;
      }
      enough = true;
    }
    wave_fence();
  }
  const int have = rank_list(list, best, n, K, lane);

  const float all = wave_max(top);
  const double total = wave_sum(top == -INFINITY ? 0.0 : sum * (double)__builtin_amdgcn_exp2f((top - all) * 1.44269504088896341f));
  uint8_t* out = work + (int64_t)id * part_bytes(K);
  if (lane == 0) *reinterpret_cast<Part*>(out) = Part{total, all, 0};
  if (lane < K) reinterpret_cast<Entry*>(out + sizeof(Part))[lane] = lane < have ? best[lane] : Entry{-INFINITY, INT_MAX};
}

// T threads: 256, or 512 where there are more than 256 lists or 1024 possible candidates.  `shift`: a row's lists lie in 2^shift lanes of one wave.
constexpr int picks_of(int threads) { return threads == 256 ? 1024 : 4096; }

template <int KMAX, int T>
__global__ __launch_bounds__(T) void beam_pick_kernel(BeamSelect a, int parts, int shift, const uint8_t* work) {
  __shared__ float bound_s[T / 64];
  __shared__ double score_s[picks_of(T)];   // candidates: the score and beam * vocab + id, below 2^28
  __shared__ int flat_s[picks_of(T)];
  __shared__ uint8_t end_s[kBeamMax];
  __shared__ int n_s;
  const int K = a.beams, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row0 = (int)blockIdx.x * K, stride = (int)part_bytes(K);
  work += (int64_t)row0 * parts * stride;
  if (threadIdx.x == 0) n_s = 0;
  // everything this workgroup reads, at once: a thread's list (beam, part), best first, and the part's sum
  const int k = min((int)threadIdx.x >> shift, K - 1), p = (int)threadIdx.x & ((1 << shift) - 1);
  const bool mine = (int)threadIdx.x >> shift < K && p < parts;
  const uint8_t* from = work + (k * parts + (mine ? p : 0)) * stride;
  const Part q = *reinterpret_cast<const Part*>(from);
  const uint4* src = reinterpret_cast<const uint4*>(from + sizeof(Part));
  Entry list[KMAX];
#pragma unroll
  for (int e = 0; e < KMAX; e += 2) {
    const uint4 u = src[min(e / 2, (K - 1) / 2)];
    list[e] = Entry{__uint_as_float(u.x), (int)u.y}, list[e + 1] = Entry{__uint_as_float(u.z), (int)u.w};
  }
  const float my_score = a.scores[row0 + k];
  const bool my_end = a.finished[row0 + k] != 0;
  if (p == 0) end_s[k] = my_end;
  // score_k - log sum exp of row k; -inf: a beam with no candidates of its own (finished, not in use).  (The differences of the parts' maxima
  // in 64 bits: far below 32 bits' rounding of the exponent.)
  const float part_top = mine && !my_end && my_score > -INFINITY ? q.top : -INFINITY;
  float top = part_top;
#pragma unroll 1
  for (int o = 0; o < shift; ++o) top = fmaxf(top, __shfl_xor(top, 1 << o));
  double sum = part_top == -INFINITY ? 0.0 : q.sum * exp((double)part_top - (double)top);
#pragma unroll 1
  for (int o = 0; o < shift; ++o) sum += __shfl_xor(sum, 1 << o);
  double offset = -INFINITY, head = -INFINITY;
  const int flat0 = k * a.vocab;
  int self = -1;   // a finished beam's first list is the beam itself
  if (mine) {
    if (my_end) {
      if (p == 0) self = flat0 + (a.eos > 0 ? a.eos : 0), head = (double)my_score;
    } else if (top > -INFINITY) {
      offset = (double)my_score - (log(sum) + (double)top);
      head = offset + (double)list[0].val;
    }
  }
  const float kth = wave_kth((float)head, K, lane);
  if (lane == 0) bound_s[wave] = kth;
  __syncthreads();
  float bound = bound_s[0];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) bound = fmaxf(bound, bound_s[w]);
  auto add = [&](double score, int flat) {   // (any order: it is ranked below)
    const int at = atomicAdd(&n_s, 1);
    score_s[at] = score, flat_s[at] = flat;
  };
  if (self >= 0) {
    if (head > -INFINITY && (float)head >= bound) add(head, self);
  } else if (offset > -INFINITY) {
#pragma unroll
    for (int e = 0; e < KMAX; ++e) {
      const double v = offset + (double)list[e].val;
      if (e < K && list[e].val > -INFINITY && (float)v >= bound) add(v, flat0 + list[e].idx);
    }
  }
  __syncthreads();
  const int n = n_s;
  auto put = [&](int slot, double score, int parent, int token, bool done) {
    a.out_scores[row0 + slot] = (float)score;
    a.parents[row0 + slot] = parent;
    a.tokens[row0 + slot] = token;
    a.out_finished[row0 + slot] = done ? 1 : 0;
  };
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += T) {
    const double score = score_s[i];
    const int flat = flat_s[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += score_s[j] > score || (score_s[j] == score && flat_s[j] < flat) ? 1 : 0;
    if (rank < K) {
      const int parent = flat / a.vocab;
      const bool over = end_s[parent] != 0;
      const int token = over ? a.eos : flat - parent * a.vocab;
      put(rank, score, parent, token, over || token == a.eos);
    }
  }
  if ((int)threadIdx.x >= n && (int)threadIdx.x < K) put(threadIdx.x, -INFINITY, threadIdx.x, a.eos, true);   // too few candidates
}

int lanes_shift(int parts) {
  int s = 0;
  while (1 << s < parts) ++s;
  return s;
}

// parts of a row: enough waves to fill the chip, at least a chunk each, and lists that pass 2 holds at one a thread
// (fixed: as for one entry, whatever the batch is)
int beam_parts(int batch, int beams, int vocab, bool fixed) {
  const int64_t rows = (int64_t)(fixed ? 1 : batch) * beams;
  int64_t n = (12288 + rows - 1) / rows;
  const int64_t chunks = (vocab + 64 * kLane - 1) / (64 * kLane);
  n = n < chunks ? n : chunks;
  const int64_t most = picks_of(512) / (beams * beams);
  n = n < most ? n : most;
  n = n < kPartsMax ? n : kPartsMax;
  n = n < 1 ? 1 : n;
  while ((beams << lanes_shift((int)n)) > 512) n = 1 << (lanes_shift((int)n) - 1);
  return (int)n;
}

template <int KMAX>
void launch_pick(const BeamSelect& a, int parts, const uint8_t* work, hipStream_t s) {
  const int shift = lanes_shift(parts);
  if (a.beams << shift <= 256 && a.beams * a.beams * parts <= picks_of(256)) MSH_LAUNCH((beam_pick_kernel<KMAX, 256>), dim3(a.batch), dim3(256), 0, s, a, parts, shift, work);
  else MSH_LAUNCH((beam_pick_kernel<KMAX, 512>), dim3(a.batch), dim3(512), 0, s, a, parts, shift, work);
}

// ---- reordering ---------------------------------------------------------------------------------------------------------
// state[b, k, :len_b] <- state[b, parent[b, k], :len_b] in place.  A thread owns one piece (16 bytes) of all beams of (outer, b, inner): it
// loads what its beams' parents have there, then stores -- no thread reads what another writes, whatever the parents are, and a beam
// that continues itself is neither read nor written.  One piece a thread: several in turn measured slower (four: 758 us instead of 238), since a
// workgroup's time is the latency of its chain of loads.  Bound by HBM bandwidth: 8 layers of 32 entries x 8 beams x 8 heads, up to 447 rows of 52 bf16
// keys and values (1.1 GB): 238 us, 4.6 TB/s; one clip's four beams after 33 steps: 7.3 us.
struct BeamStates {
  BeamState s[kBeamStates];
  uint32_t first[kBeamStates];      // first workgroup of each state
  uint32_t blocks[kBeamStates];     // workgroups of one (outer, b, inner)
  int32_t unit[kBeamStates];        // bytes of a piece: 16, 4 or 1, as the state's address and strides allow
};

// from[k]: the beam to read for beam k -- for a beam that stays one that is read anyway, so that no load hangs on a condition (each would be
// waited for where its condition ends); move: bit k = beam k is written
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));   // (an array of HIP's uint4 class ends up in scratch memory: twice the writes)
template <int KMAX, class P>
__device__ __forceinline__ void move_piece(uint8_t* p, int64_t stride, const int32_t* from, uint32_t move) {
  P v[KMAX];
#pragma unroll
  for (int k = 0; k < KMAX; ++k) v[k] = *reinterpret_cast<const P*>(p + from[k] * stride);
#pragma unroll
  for (int k = 0; k < KMAX; ++k)
    if ((move >> k) & 1) *reinterpret_cast<P*>(p + k * stride) = v[k];
}

template <int KMAX>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamStates all, int n_states, uint32_t batch, int beams, const int32_t* parents,
                                                           const int32_t* lengths, int length_stride) {
  BeamState s = all.s[0];
  uint32_t first = 0, blocks = all.blocks[0];
  int unit = all.unit[0];
#pragma unroll
  for (int i = 1; i < kBeamStates; ++i)
    if (i < n_states && blockIdx.x >= all.first[i]) s = all.s[i], first = all.first[i], blocks = all.blocks[i], unit = all.unit[i];
  const uint32_t at = blockIdx.x - first, seg = at / blocks, slice = at - seg * blocks;
  const uint32_t n_inner = (uint32_t)s.inner, rest = seg / n_inner, inner = seg - rest * n_inner, outer = rest / batch, b = rest - outer * batch;
  const int32_t* par = parents + (int64_t)b * beams;
  const int32_t given = *(lengths != nullptr ? lengths + (int64_t)b * length_stride : par);
  int32_t f[KMAX], from[KMAX];
#pragma unroll
  for (int k = 0; k < KMAX; ++k) f[k] = par[k < beams ? k : beams - 1];
  int64_t rows = lengths != nullptr ? given : s.n_rows;
  rows = rows < 0 ? 0 : rows > s.n_rows ? s.n_rows : rows;
  const int64_t bytes = rows * s.row_bytes;
  const int64_t o = (int64_t)slice * 256 * unit + (int64_t)threadIdx.x * unit;
  uint32_t move = 0;
  int32_t some = 0;
#pragma unroll
  for (int k = 0; k < KMAX; ++k)
    if (k < beams && f[k] != k && f[k] >= 0 && f[k] < beams) move |= 1u << k, some = f[k];
  if (move == 0 || o >= bytes) return;
#pragma unroll
  for (int k = 0; k < KMAX; ++k) from[k] = (move >> k) & 1 ? f[k] : some;
  uint8_t* p = static_cast<uint8_t*>(s.data) + outer * s.outer_stride + b * (beams * s.beam_stride) + inner * s.inner_stride;
  const int64_t stride = s.beam_stride;
  if (o + unit <= bytes && unit == 16) {
    move_piece<KMAX, u32x4>(p + o, stride, from, move);
  } else if (o + unit <= bytes && unit == 4) {
    move_piece<KMAX, uint32_t>(p + o, stride, from, move);
  } else {   // single bytes, and the last piece of the valid rows
#pragma unroll 1
    for (int64_t c = o; c < o + unit && c < bytes; ++c) move_piece<KMAX, uint8_t>(p + c, stride, from, move);
  }
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

size_t beam_select_work_bytes(int batch, int beams, int vocab, bool fixed) {
  return (size_t)batch * beams * beam_parts(batch, beams, vocab, fixed) * part_bytes(beams);
}

void beam_select(const BeamSelect& a, Elem type, hipStream_t s) {
  const int parts = beam_parts(a.batch, a.beams, a.vocab, a.fixed);
  const dim3 grid((unsigned)(((int64_t)a.batch * a.beams * parts + 3) / 4));
  uint8_t* work = static_cast<uint8_t*>(a.work);
  if (type == Elem::f32) MSH_LAUNCH((beam_partial_kernel<Elem::f32>), grid, dim3(256), 0, s, a, parts, work);
  else if (type == Elem::bf16) MSH_LAUNCH((beam_partial_kernel<Elem::bf16>), grid, dim3(256), 0, s, a, parts, work);
  else MSH_LAUNCH((beam_partial_kernel<Elem::f16>), grid, dim3(256), 0, s, a, parts, work);
  if (a.beams <= 4) launch_pick<4>(a, parts, work, s);
  else if (a.beams <= 8) launch_pick<8>(a, parts, work, s);
  else launch_pick<16>(a, parts, work, s);
}

static int64_t piece_bytes(const BeamState& st) {
  auto fits = [&](int64_t u) {
    return (uintptr_t)st.data % u == 0 && (st.outer == 1 || st.outer_stride % u == 0) && st.beam_stride % u == 0 &&
           (st.inner == 1 || st.inner_stride % u == 0);
  };
  return fits(16) ? 16 : fits(4) ? 4 : 1;
}
int64_t beam_reorder_groups(const BeamState* states, int n_states, int batch) {
  int64_t n = 0;
  for (int i = 0; i < n_states; ++i) {
    const int64_t bytes = states[i].n_rows * states[i].row_bytes, slice = 256 * piece_bytes(states[i]);
    n += states[i].outer * batch * states[i].inner * ((bytes + slice - 1) / slice);
  }
  return n;
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
    const int64_t unit = piece_bytes(st), slice = 256 * unit;
    all.s[n] = st;
    all.first[n] = (uint32_t)blocks;
    all.unit[n] = (int32_t)unit;
    all.blocks[n] = (uint32_t)((bytes + slice - 1) / slice);
    blocks += st.outer * batch * st.inner * all.blocks[n];
    ++n;
  }
  if (n == 0 || beams < 2) return;
  const dim3 grid((unsigned)blocks);
  if (beams <= 4) MSH_LAUNCH(beam_reorder_kernel<4>, grid, dim3(256), 0, s, all, n, (uint32_t)batch, beams, parents, lengths, length_stride);
  else if (beams <= 8) MSH_LAUNCH(beam_reorder_kernel<8>, grid, dim3(256), 0, s, all, n, (uint32_t)batch, beams, parents, lengths, length_stride);
  else MSH_LAUNCH(beam_reorder_kernel<16>, grid, dim3(256), 0, s, all, n, (uint32_t)batch, beams, parents, lengths, length_stride);
}

}  // namespace msh
