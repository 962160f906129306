// Attention over the paged 4-bit cache (form: serve_kernels.h), one instantiation per element type (k_kv4_{f32,bf16,f16}.hip).
//
//   out[r, h] = sum_t p_t V_t,  p = softmax over the visible t of scale * q[r, h] . K_t
//
// A wave takes 16 * RT query rows of one key / value head -- the rows of all query heads that share it and of all tokens of the call --
// and walks blocks of 32 cached tokens:
//   S^T = K q^T    16x16x32 per (16 tokens, group): A = the block's bytes as they lie, expanded to bf16 by the conversion that applies
//                  the power of two (exact), B = the rows' q, held in registers for the whole walk
//   O^T += V^T P^T per (16 elements, 32 tokens): the accumulators of S^T already lie in the order the B operand wants (lane = 16 *
//                  quarter + row; its eight tokens are 4 * quarter + {0..3} of both 16-token tiles), and the values' bytes are laid out
//                  for that order: P never leaves the lane.  A byte holds two elements of one token, so the expansion gives
//                  {even, odd} pairs, and one byte permutation per pair of tokens makes the operands of an even and an odd tile.
// No shared memory and no barrier in the walk; the next block's bytes are in flight while this one is computed.
//
// Exactness: the cached values are exact in bf16.  q of fp16 / fp32 is the sum of 2 / 3 bf16 terms, p of 2 (3 for fp32 outputs) terms;
// products, softmax statistics and sums are fp32.  The running maximum follows only when a score passes it by 2^8 (log2 units: 8), so
// the common block needs no cross-lane step and no rescaling; p <= 2^8 keeps its relative precision.
#pragma once

#include "kernels.h"
#include "kv4_common.h"

namespace msh {
namespace {

template <Elem E>
struct Terms;   // bf16 terms of a query element and of a probability
template <>
struct Terms<Elem::bf16> { static constexpr int q = 1, p = 2; };
template <>
struct Terms<Elem::f16> { static constexpr int q = 2, p = 2; };
template <>
struct Terms<Elem::f32> { static constexpr int q = 3, p = 3; };

union Frag {
  uint32_t u[4];
  bf16x8 v;
};

template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t* out) {
  if constexpr (N >= 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    out[0] = x.x, out[1] = x.y, out[2] = x.z, out[3] = x.w;
    if constexpr (N > 4) load_dwords<N - 4>(p + 16, out + 4);
  } else if constexpr (N == 3) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    out[0] = w[0], out[1] = w[1], out[2] = w[2];
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    out[0] = x.x, out[1] = x.y;
  } else if constexpr (N == 1) {
    out[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// one block's bytes of a lane
template <int M>
struct BlockBytes {
  uint32_t k[2][M], ks[2][(M + 3) / 4], v[2 * M], vs[2 * M];

  __device__ __forceinline__ void load(const uint8_t* b, int lane) {
    const int quarter = lane >> 4, idx = lane & 15;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const uint8_t* p = b + tile * 256 * M;
      if constexpr (M <= 4) {
        load_dwords<M>(p + lane * 4 * M, k[tile]);
      } else {
        load_dwords<4>(p + lane * 16, k[tile]);
        load_dwords<M - 4>(p + 1024 + lane * 4 * (M - 4), k[tile] + 4);
      }
      const uint8_t* q = b + 512 * M + (tile * 16 + idx) * M;
      if constexpr (M % 4 == 0) {
#pragma unroll
        for (int i = 0; i < M / 4; ++i) ks[tile][i] = reinterpret_cast<const uint32_t*>(q)[i];
      } else if constexpr (M % 2 == 0) {
#pragma unroll
        for (int i = 0; i < (M + 3) / 4; ++i) ks[tile][i] = 0;
#pragma unroll
        for (int i = 0; i < M / 2; ++i) ks[tile][i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(q)[i] << (16 * (i & 1));
      } else {
#pragma unroll
        for (int i = 0; i < (M + 3) / 4; ++i) ks[tile][i] = 0;
#pragma unroll
        for (int i = 0; i < M; ++i) ks[tile][i / 4] |= (uint32_t)q[i] << (8 * (i & 3));
      }
    }
    const uint8_t* p = b + 544 * M;
#pragma unroll
    for (int c = 0; c < M / 2; ++c) load_dwords<4>(p + c * 1024 + lane * 16, v + 4 * c);
    if constexpr (M % 2 == 1) load_dwords<2>(p + (M / 2) * 1024 + lane * 8, v + 2 * (M - 1));
    const uint8_t* s = b + 1056 * M + quarter * 8 * M;
    if constexpr (M % 2 == 0) {
#pragma unroll
      for (int i = 0; i < M / 2; ++i) load_dwords<4>(s + 16 * i, vs + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < M; ++i) load_dwords<2>(s + 8 * i, vs + 2 * i);
    }
  }
};

__device__ __forceinline__ Frag expand_keys(uint32_t codes, uint32_t scales, int byte) {   // (byte: a constant after unrolling)
  const float s = byte == 0 ? kv4_scale_of<0>(scales) : byte == 1 ? kv4_scale_of<1>(scales) : byte == 2 ? kv4_scale_of<2>(scales) : kv4_scale_of<3>(scales);
  Frag f;
  f.u[0] = kv4_pair_bf16<0>(codes, s);
  f.u[1] = kv4_pair_bf16<1>(codes, s);
  f.u[2] = kv4_pair_bf16<2>(codes, s);
  f.u[3] = kv4_pair_bf16<3>(codes, s);
  return f;
}

// eight tokens x {even, odd} element -> the operands of the even and the odd tile
__device__ __forceinline__ void expand_values(const uint32_t* v, const uint32_t* vs, Frag& even, Frag& odd) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t c = v[half], s = vs[half];
    const uint32_t t0 = kv4_pair_bf16<0>(c, kv4_scale_of<0>(s)), t1 = kv4_pair_bf16<1>(c, kv4_scale_of<1>(s));
    const uint32_t t2 = kv4_pair_bf16<2>(c, kv4_scale_of<2>(s)), t3 = kv4_pair_bf16<3>(c, kv4_scale_of<3>(s));
    even.u[2 * half] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
    odd.u[2 * half] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
    even.u[2 * half + 1] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
    odd.u[2 * half + 1] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
  }
}

// x (replaced by what is left) -> its leading bf16 term, eight at a time
__device__ __forceinline__ Frag take_term(float* x, bool rest) {
  Frag f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.u[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    if (rest) {
      x[2 * i] -= __uint_as_float(f.u[i] << 16);
      x[2 * i + 1] -= __uint_as_float(f.u[i] & 0xffff0000u);
    }
  }
  return f;
}

__device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}

// The walk of one wave: RT tiles of 16 query rows of key / value head `head`.
template <int M, Elem E, int RT>
struct Walk {
  static constexpr int QT = Terms<E>::q, PT = Terms<E>::p;
  Frag q[RT][M][QT];
  f32x4 acc[RT][2 * M];   // [2 g + parity]: elements 32 g + 8 quarter + 2 r + parity of row idx
  float top[RT], sum[RT]; // sum: of this lane's tokens only
  int last[RT];           // last visible token of this lane's row (causal), first visible
  int low[RT];

  // plain: every row sees all 32 tokens (uniform).  The empty asm keeps the masks behind their branch -- they would be computed for every
  // block otherwise --; a second copy of the step costs more registers than it saves
  __device__ __forceinline__ void step(const BlockBytes<M>& b, int t0, int len, bool plain, float scale_log2, int quarter) {
    f32x4 s[RT][2];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][tile] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < M; ++g) {
        const Frag k = expand_keys(b.k[tile][g], b.ks[tile][g / 4], g & 3);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int w = QT - 1; w >= 0; --w) s[rt][tile] = mma(k, q[rt][g][w], s[rt][tile]);   // small terms first
      }
    }
    uint32_t keep[2] = {~0u, ~0u};   // bytes of the tokens that exist, of this lane's 4 + 4
    if (!plain) {
      asm volatile("" ::: );
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        keep[half] = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (t0 + half * 16 + quarter * 4 + c < len) keep[half] |= 255u << (8 * c);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = t0 + (e >> 2) * 16 + quarter * 4 + (e & 3);
          s[rt][e >> 2][e & 3] = t <= last[rt] && t >= low[rt] ? s[rt][e >> 2][e & 3] : -INFINITY;
        }
    }
    Frag p[RT][PT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8];   // q . k (times the scale's sign)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[rt][e >> 2][e & 3];
      }
      float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      hi *= scale_log2;
      if (__builtin_amdgcn_ballot_w64(hi > top[rt] + 8.f) != 0) {   // (top = -inf: any finite score)
        hi = fmaxf(hi, __shfl_xor(hi, 16));
        hi = fmaxf(hi, __shfl_xor(hi, 32));
        const float now = fmaxf(hi, top[rt]);
        const float f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[rt] - now);
        top[rt] = now;
        sum[rt] *= f;
#pragma unroll
        for (int i = 0; i < 2 * M; ++i) acc[rt][i] = acc[rt][i] * f;
      }
      const float ref = top[rt] == -INFINITY ? 0.f : top[rt];
      float add = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], scale_log2, -ref));
        add += x[e];
      }
      sum[rt] += add;
#pragma unroll
      for (int w = 0; w < PT; ++w) p[rt][w] = take_term(x, w + 1 < PT);
    }
#pragma unroll
    for (int g = 0; g < M; ++g) {
      uint32_t vs[2] = {b.vs[2 * g], b.vs[2 * g + 1]};
      if (!plain) {   // a token past the end: whatever its scale byte is, 0 * finite = 0
        asm volatile("" ::: );
#pragma unroll
        for (int half = 0; half < 2; ++half) vs[half] = (vs[half] & keep[half]) | (0x7f7f7f7fu & ~keep[half]);
      }
      Frag even, odd;
      expand_values(b.v + 2 * g, vs, even, odd);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int w = PT - 1; w >= 0; --w) {
          acc[rt][2 * g] = mma(even, p[rt][w], acc[rt][2 * g]);
          acc[rt][2 * g + 1] = mma(odd, p[rt][w], acc[rt][2 * g + 1]);
        }
    }
  }
};

// KW: waves that share 16 * RT rows, take the blocks of the workgroup's range in turn and join their results in shared memory; 4 / KW such
//   units (a tile of rows of a sequence and key / value head) make a workgroup.  KW = 4 where few rows have long caches, 1 where there
//   are rows enough -- chunks of prompts, many short sequences --: a wave's beginning and end cost as much as three blocks.
// waves per SIMD: left alone the compiler spends the registers of two or three waves on one; asked for more it spills
template <int M, Elem E, int RT>
constexpr int waves_wanted() {
  if (RT == 1) return M <= 2 ? 4 : M <= 4 && E != Elem::f32 ? 3 : 2;
  return M <= 2 ? (E == Elem::bf16 ? 3 : 2) : M <= 4 && E != Elem::f32 ? 2 : 1;
}
template <int M, Elem E, int RT, int KW>
__global__ __launch_bounds__(256, (waves_wanted<M, E, RT>())) void kv4_attention_kernel(Kv4Attention a) {
  typedef typename ElemOf<E>::T T;
  constexpr int DP = 32 * M;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int quarter = lane >> 4, idx = lane & 15;
  const int heads_kv = a.cache.heads, per = a.heads / heads_kv;
  // unit = ((sequence, key / value head), tile of rows); the second grid axis is the key range
  const int sub = wave % KW, unit = (int)blockIdx.x * (4 / KW) + wave / KW, split = blockIdx.y;
  const int pair = unit / a.tiles, tile0 = unit - pair * a.tiles;
  int b = pair / heads_kv;
  const int head = pair - b * heads_kv;
  bool active = b < a.batch;   // (a wave without work stays for the barriers of its workgroup)
  b = active ? b : 0;
  const int page_shift = a.cache.page_shift;
  const int64_t q0 = a.q_start != nullptr ? a.q_start[b] : (int64_t)b * a.max_q;
  int n_q = a.q_start != nullptr ? a.q_start[b + 1] - a.q_start[b] : a.max_q;
  if (n_q > a.max_q) n_q = a.max_q;
  active = active && q0 >= 0 && n_q > 0 && q0 + n_q <= a.rows;   // (a q_start that does not fit: nothing is written)
  const int n_rows = active ? n_q * per : 0;
  const int row0 = tile0 * 16 * RT;
  active = active && row0 < n_rows;
  if (KW == 1 && !active) return;
  int len = a.kv_lens[b];
  const int64_t room = (int64_t)a.width << page_shift;
  len = len < 0 ? 0 : len > room ? (int)room : len;

  Walk<M, E, RT> w;
  int64_t row_of[RT];   // query row of this lane's column, its query head; -1: none
  int head_of[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + idx;
    const int tq = r / per, g = r % per;
    const bool there = r < n_rows;
    row_of[rt] = there ? q0 + tq : -1;
    head_of[rt] = there ? head * per + g : head * per;
    const int at = len - n_q + tq;   // place of the query's own token
    w.last[rt] = !there ? -1 : a.causal ? at : len - 1;
    if (w.last[rt] >= len) w.last[rt] = len - 1;
    w.low[rt] = a.causal && a.window > 0 ? at - a.window + 1 : 0;
    w.top[rt] = -INFINITY, w.sum[rt] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) w.acc[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // every load is issued whatever the lane's row and element are (clamped into the row, selected afterwards): a load behind a
    // condition of its own waits for the one before it
    const T* src = static_cast<const T*>(a.q) + (there ? row_of[rt] : active ? q0 : 0) * a.q_row + head_of[rt] * a.q_head;
    float x[M][8];
    if (a.vec) {
#pragma unroll
      for (int g2 = 0; g2 < M; ++g2)
#pragma unroll
        for (int c = 0; c < 8; c += 4) {
          const int d = g2 * 32 + quarter * 8 + c;
          load_elems<E, 4>(src + (d + 4 <= a.cache.head_dim ? d : a.cache.head_dim - 4), &x[g2][c]);
        }
    } else {
#pragma unroll
      for (int g2 = 0; g2 < M; ++g2)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = g2 * 32 + quarter * 8 + e;
          x[g2][e] = ElemOf<E>::get(src[d < a.cache.head_dim ? d : a.cache.head_dim - 1]);
        }
    }
#pragma unroll
    for (int g2 = 0; g2 < M; ++g2) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[g2][e] = there && g2 * 32 + quarter * 8 + e < a.cache.head_dim ? x[g2][e] * a.sign : 0.f;
#pragma unroll
      for (int t = 0; t < Walk<M, E, RT>::QT; ++t) w.q[rt][g2][t] = take_term(x[g2], t + 1 < Walk<M, E, RT>::QT);
    }
  }

  // tokens that some row of the tile sees: [from, to); [all_from, all_to): that every row sees
  const int tq0 = row0 / per, tq1 = (row0 + 16 * RT < n_rows ? row0 + 16 * RT - 1 : n_rows - 1) / per;
  int to = a.causal ? len - n_q + tq1 + 1 : len, all_to = a.causal ? len - n_q + tq0 + 1 : len;
  to = to < 0 ? 0 : to;
  int from = 0, all_from = 0;
  if (a.causal && a.window > 0) {
    from = len - n_q + tq0 - a.window + 1, all_from = len - n_q + tq1 - a.window + 1;
    from = from < 0 ? 0 : from;
  }
  int blk0 = from >> 5, blk1 = (to + 31) >> 5;
  if (a.nsplit > 1) {
    const int n = blk1 - blk0, share = (n + a.nsplit - 1) / a.nsplit;
    const int s0 = blk0 + split * share;
    blk1 = s0 + share < blk1 ? s0 + share : blk1;
    blk0 = s0;
  }
  if (!active) blk1 = blk0;
  const int32_t* table = a.table + (int64_t)b * a.width;
  const int64_t block_bytes = kv4_block_bytes(M);
  const int in_shift = page_shift - 5, in_mask = (1 << in_shift) - 1;
  // (blocks behind the last are the last again, and a page that is not in the cache is page 0, not looked at: the loads of a step are
  // unconditional, or each would be waited for where its condition ends)
  auto page_of = [&](int blk) -> int32_t { return table[(blk < blk1 ? blk : blk1 - 1) >> in_shift]; };
  auto good = [&](int32_t page) { return page >= 0 && page < a.cache.pages; };
  auto at = [&](int blk, int32_t page) {
    return a.cache.data + ((((int64_t)(good(page) ? page : 0) * heads_kv + head) << in_shift) + ((blk < blk1 ? blk : blk1 - 1) & in_mask)) * block_bytes;
  };
  auto plain = [&](int blk) { return blk * 32 >= all_from && blk * 32 + 32 <= all_to && blk * 32 + 32 <= len; };

  constexpr int step = KW;
  int blk = blk0 + sub;
  if (blk < blk1) {
    BlockBytes<M> x, y;
    int32_t px = page_of(blk), py = page_of(blk + step);
    auto walk = [&](const BlockBytes<M>& bytes) { w.step(bytes, blk * 32, len, plain(blk), a.scale_log2, quarter); };
    x.load(at(blk, px), lane);
    while (true) {
      const int32_t next = page_of(blk + 2 * step);
      y.load(at(blk + step, py), lane);
      if (good(px)) walk(x);
      blk += step;
      if (blk >= blk1) break;
      px = next;
      const int32_t after = page_of(blk + 2 * step);
      x.load(at(blk + step, px), lane);
      if (good(py)) walk(y);
      blk += step;
      if (blk >= blk1) break;
      py = after;
    }
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    w.sum[rt] += __shfl_xor(w.sum[rt], 16);
    w.sum[rt] += __shfl_xor(w.sum[rt], 32);
  }

  auto finish = [&](int64_t row, int h, int d0, const float* v, float top, float sum, bool first) {   // eight elements from d0 on
    if (a.nsplit > 1) {
      float* p = a.part + ((row * a.heads + h) * a.nsplit + split) * (DP + kPartPad);
      *reinterpret_cast<float4*>(p + d0) = float4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<float4*>(p + d0 + 4) = float4{v[4], v[5], v[6], v[7]};
      if (first) p[DP] = top, p[DP + 1] = sum;
      return;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v[e] * inv;
    if (a.fm != nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < a.cache.head_dim) a.fm[fm16((int)row, h * a.cache.head_dim + d0 + e, a.heads * a.cache.head_dim >> 5)] = ElemOf<Elem::bf16>::put(x[e]);
      return;
    }
    T* o = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head + d0;
    if (a.vec) {
      if (d0 + 4 <= a.cache.head_dim) store_elems<E, 4>(o, x);
      if (d0 + 8 <= a.cache.head_dim) store_elems<E, 4>(o + 4, x + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < a.cache.head_dim) o[e] = ElemOf<E>::put(x[e]);
    }
    if (first && a.lse != nullptr) a.lse[row * a.heads + h] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f : -INFINITY;
  };

  if constexpr (KW == 1) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (row_of[rt] < 0) continue;
#pragma unroll
      for (int g = 0; g < M; ++g) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[2 * r] = w.acc[rt][2 * g][r], v[2 * r + 1] = w.acc[rt][2 * g + 1][r];
        finish(row_of[rt], head_of[rt], g * 32 + quarter * 8, v, w.top[rt], w.sum[rt], g == 0 && quarter == 0);
      }
    }
  } else {
    constexpr int LD = DP + 4;   // (16 rows' 16-byte pieces spread over the banks)
    __shared__ float part[4][16][LD];
    __shared__ float stat[4][16][2];
    const int first_wave = wave - sub;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (rt > 0) __syncthreads();
      if (quarter == 0) stat[wave][idx][0] = w.top[rt], stat[wave][idx][1] = w.sum[rt];
#pragma unroll
      for (int g = 0; g < M; ++g) {
        float4 lo{w.acc[rt][2 * g][0], w.acc[rt][2 * g + 1][0], w.acc[rt][2 * g][1], w.acc[rt][2 * g + 1][1]};
        float4 hi{w.acc[rt][2 * g][2], w.acc[rt][2 * g + 1][2], w.acc[rt][2 * g][3], w.acc[rt][2 * g + 1][3]};
        *reinterpret_cast<float4*>(&part[wave][idx][g * 32 + quarter * 8]) = lo;
        *reinterpret_cast<float4*>(&part[wave][idx][g * 32 + quarter * 8 + 4]) = hi;
      }
      __syncthreads();
      for (int i = sub * 64 + lane; i < 16 * 4 * M; i += KW * 64) {
        const int col = i / (4 * M), d0 = (i % (4 * M)) * 8, r = row0 + rt * 16 + col;
        if (r >= n_rows) continue;
        float top = stat[first_wave][col][0];
#pragma unroll
        for (int v = 1; v < KW; ++v) top = fmaxf(top, stat[first_wave + v][col][0]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < KW; ++v) {
          const float f = __builtin_amdgcn_exp2f(stat[first_wave + v][col][0] - ref);
          sum += stat[first_wave + v][col][1] * f;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += part[first_wave + v][col][d0 + e] * f;
        }
        finish(q0 + r / per, head * per + r % per, d0, o, top, sum, d0 == 0);
      }
    }
  }
}

// joins the key ranges of one (row, head): one wave each
template <Elem E>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4Attention a, int dp) {
  typedef typename ElemOf<E>::T T;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = id / a.heads;
  const int h = (int)(id % a.heads);
  if (row >= a.rows) return;
  int b;   // rows that no sequence owns are left as they are
  if (a.q_start != nullptr) {
    int lo = 0, hi = a.batch;
    while (lo < hi) {   // last sequence that starts at or before the row
      const int mid = (lo + hi + 1) >> 1;
      if (mid < a.batch && a.q_start[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    const int64_t q0 = a.q_start[b], q1 = a.q_start[b + 1];
    if (row < q0 || row >= q1 || row >= q0 + a.max_q || q0 < 0 || (q1 - q0 > a.max_q ? q0 + a.max_q : q1) > a.rows) return;
  } else if (row >= (int64_t)a.batch * a.max_q) {
    return;
  }
  // lane s: the maximum and the sum of range s (at most 64 of them)
  const int64_t stride = dp + kPartPad;
  const float* p = a.part + (row * a.heads + h) * a.nsplit * stride;
  float mine = -INFINITY, part_sum = 0.f;
  if (lane < a.nsplit) mine = p[lane * stride + dp], part_sum = p[lane * stride + dp + 1];
  float top = mine;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - top);
  float sum = part_sum * f;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  T* o = static_cast<T*>(a.out) + row * a.out_row + h * a.out_head;
  // a lane has four elements; where those take up half the wave or less, groups of lanes take the ranges in turn: all rows are in flight at once
  const int per = dp >> 2, groups = 64 / per, group = lane / per, d0 = (lane - group * per) * 4;
  float4 v{0.f, 0.f, 0.f, 0.f};
  if (group < groups) {
#pragma unroll 8
    for (int s = group; s < a.nsplit; s += groups) {
      const float4 x = *reinterpret_cast<const float4*>(p + s * stride + d0);
      const float g = __shfl(f, s);
      v.x += x.x * g, v.y += x.y * g, v.z += x.z * g, v.w += x.w * g;
    }
  }
  for (int k = 1; k < groups; ++k) {
    const float4 x{__shfl(v.x, lane + k * per), __shfl(v.y, lane + k * per), __shfl(v.z, lane + k * per), __shfl(v.w, lane + k * per)};
    if (group == 0) v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
  }
  if (group == 0) {
    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = d0 + e;
      if (d >= a.cache.head_dim) break;
      if (a.fm != nullptr) a.fm[fm16((int)row, h * a.cache.head_dim + d, a.heads * a.cache.head_dim >> 5)] = ElemOf<Elem::bf16>::put(y[e]);
      else o[d] = ElemOf<E>::put(y[e]);
    }
  }
  if (lane == 0 && a.lse != nullptr) a.lse[row * a.heads + h] = sum > 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f : -INFINITY;
}

template <int M, Elem E>
void launch_kv4_attention(const Kv4Attention& a0, hipStream_t s) {
  Kv4Attention a = a0;
  const Kv4Shape shape = kv4_attention_shape(a);
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads);
  const int64_t pairs = (int64_t)a.batch * a.cache.heads;
  a.tiles = (int32_t)((rows + 16 * shape.rt - 1) / (16 * shape.rt));
  const int64_t four = E == Elem::f32 ? 16 : 8;   // bytes of four elements
  const int64_t size = four / 4;
  auto even = [&](const void* p, int64_t row, int64_t head) { return (uintptr_t)p % four == 0 && row * size % four == 0 && head * size % four == 0; };
  a.vec = a.cache.head_dim % 4 == 0 && even(a.q, a.q_row, a.q_head) && (a.fm != nullptr || even(a.out, a.out_row, a.out_head));
  a.sign = a.scale_log2 < 0.f ? -1.f : 1.f;
  a.scale_log2 = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);   // (0 * -inf of a masked score would be NaN; any score times this is 0 to exp2)
  const int64_t per_group = 4 / shape.kw;
  const dim3 grid((unsigned)((pairs * a.tiles + per_group - 1) / per_group), (unsigned)a.nsplit);
  if (shape.rt == 1 && shape.kw == 4) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 4>), grid, dim3(256), 0, s, a);
  else if (shape.rt == 1 && shape.kw == 2) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 2>), grid, dim3(256), 0, s, a);
  else if (shape.rt == 1) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 1>), grid, dim3(256), 0, s, a);
  else if (shape.kw == 4) MSH_LAUNCH((kv4_attention_kernel<M, E, 2, 4>), grid, dim3(256), 0, s, a);
  else MSH_LAUNCH((kv4_attention_kernel<M, E, 2, 1>), grid, dim3(256), 0, s, a);
  if (a.nsplit > 1) MSH_LAUNCH((kv4_join_kernel<E>), dim3((unsigned)((a.rows * a.heads + 3) / 4)), dim3(256), 0, s, a, 32 * M);
}

template <Elem E>
void dispatch_kv4_attention(const Kv4Attention& a, hipStream_t s) {
  switch (kv4_groups(a.cache.head_dim)) {
    case 1: return launch_kv4_attention<1, E>(a, s);
    case 2: return launch_kv4_attention<2, E>(a, s);
    case 3: return launch_kv4_attention<3, E>(a, s);
    case 4: return launch_kv4_attention<4, E>(a, s);
    case 5: return launch_kv4_attention<5, E>(a, s);
    case 6: return launch_kv4_attention<6, E>(a, s);
    case 7: return launch_kv4_attention<7, E>(a, s);
    case 8: return launch_kv4_attention<8, E>(a, s);
    default: throw std::invalid_argument("kv4_attention: head width above 256");
  }
}

}  // namespace
}  // namespace msh
