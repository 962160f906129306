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
// No shared memory and no barrier in the walk; the next block's bytes are in flight while this one is computed.  (Batches of prompts have a form
// of their own, below.)
// 16 sequences of 12001 to 40000 tokens, 32 over 8 heads of 128, single bf16 tokens: 99 us and 5 for the join; the cache's 452 MB at 4.5 TB/s, HBM
// bandwidth.  256 clips of 199 to 415 frames, 8 heads of 52, four fp32 beams each: 18.8 us for 43 MB.  No unit is full (vector unit 39 % busy, the matrix unit's
// 24 products a block come to a fifth of the time): it is a wave's chain of dependent products, three for each operand, the softmax between them, and its
// beginning and end beside five or six blocks, in tiles of which 12 of 16 rows are empty.  One row a clip takes as long (18.4 us).  One clip: 7.2 us, the
// latency of a launch, of the table, the bytes and 4 blocks a wave.
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

// values' scales of tokens that do not exist: whatever the byte is, 0 * finite = 0
__device__ __forceinline__ uint32_t keep_scales(uint32_t scales, uint32_t keep) { return (scales & keep) | (0x7f7f7f7fu & ~keep); }

// keep[half]: the bytes of a lane's tokens half * 16 + quarter * 4 + 0 .. 3 of which a block of `left` tokens has
__device__ __forceinline__ void keep_of(uint32_t* keep, int left, int quarter) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    keep[half] = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (half * 16 + quarter * 4 + c < left) keep[half] |= 255u << (8 * c);
  }
}

// one block's bytes of a lane
template <int M>
struct BlockBytes {
  uint32_t k[2][M], ks[2][(M + 3) / 4], v[2 * M], vs[2 * M];

  __device__ __forceinline__ Frag keys(int tile, int g) const { return expand_keys(k[tile][g], ks[tile][g / 4], g & 3); }
  __device__ __forceinline__ void values(int g, bool plain, const uint32_t* keep, Frag& even, Frag& odd) const {
    uint32_t s[2] = {vs[2 * g], vs[2 * g + 1]};
    if (!plain) {
      asm volatile("" ::: );
      s[0] = keep_scales(s[0], keep[0]), s[1] = keep_scales(s[1], keep[1]);
    }
    expand_values(v + 2 * g, s, even, odd);
  }
  // (A uniform address and 32-bit offsets of the lane: one register an offset, no 64-bit additions.  The empty asm keeps the compiler from widening them
  // outside of the loop.)
  __device__ __forceinline__ void load(const uint8_t* b, int lane) {
    uint32_t quarter = (uint32_t)lane >> 4, idx = lane & 15, lane4 = lane * 4;
    asm("" : "+v"(quarter));
    asm("" : "+v"(idx));
    asm("" : "+v"(lane4));
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      if constexpr (M <= 4) {
        load_dwords<M>(b + lane4 * M + tile * 256 * M, k[tile]);
      } else {
        load_dwords<4>(b + lane4 * 4 + tile * 256 * M, k[tile]);
        load_dwords<M - 4>(b + lane4 * (M - 4) + (tile * 256 * M + 1024), k[tile] + 4);
      }
      const uint8_t* q = b + idx * M + (512 + tile * 16) * M;
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
#pragma unroll
    for (int c = 0; c < M / 2; ++c) load_dwords<4>(b + lane4 * 4 + (544 * M + c * 1024), v + 4 * c);
    if constexpr (M % 2 == 1) load_dwords<2>(b + lane4 * 2 + (544 * M + M / 2 * 1024), v + 2 * (M - 1));
#pragma unroll
    for (int i = 0; i < M; i += 2) {
      if constexpr (M % 2 == 0) {
        load_dwords<4>(b + quarter * 8 * M + (1056 * M + 8 * i), vs + 2 * i);
      } else {
        load_dwords<2>(b + quarter * 8 * M + (1056 * M + 8 * i), vs + 2 * i);
        if (i + 1 < M) load_dwords<2>(b + quarter * 8 * M + (1056 * M + 8 * i + 8), vs + 2 * i + 2);
      }
    }
  }
};

// x, y (replaced by what is left) -> their leading bf16 terms
__device__ __forceinline__ uint32_t take_pair(float& x, float& y, bool rest) {
  const uint32_t u = pack_bf16x2(x, y);
  if (rest) x -= __uint_as_float(u << 16), y -= __uint_as_float(u & 0xffff0000u);
  return u;
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
  int last[RT];           // last visible token of this lane's row; -1: none, or no row

  // rows row0 ... of the sequence's n_rows (row r: token r / per, head r % per of the key / value head's)
  __device__ __forceinline__ void begin(const Kv4Attention& a, int row0, int n_rows, int n_q, int len, int64_t q0, int head, int per, int quarter, int idx) {
    typedef typename ElemOf<E>::T T;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + rt * 16 + idx;
      const int tq = r / per, g = r % per;
      const bool there = r < n_rows;
      last[rt] = !there ? -1 : a.causal ? len - n_q + tq : len - 1;   // (causal: the query's own token)
      top[rt] = -INFINITY, sum[rt] = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * M; ++i) acc[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      // every load is issued whatever the lane's row and element are (clamped into the row, selected afterwards): a load behind a
      // condition of its own waits for the one before it
      const T* src = static_cast<const T*>(a.q) + (there ? q0 + tq : q0) * a.q_row + (head * per + (there ? g : 0)) * a.q_head;
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
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) q[rt][g2][t].u[i] = take_pair(x[g2][2 * i], x[g2][2 * i + 1], t + 1 < QT);
      }
    }
  }

  // s[rt][tile][c] = k[token tile * 16 + quarter * 4 + c] . q[row idx of tile rt], without the scale
  template <class Block>
  __device__ __forceinline__ void scores(const Block& b, f32x4 (&s)[RT][2]) const {
#pragma unroll
    for (int tile = 0; tile < 2; ++tile)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][tile] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < M; ++g) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const Frag k = b.keys(tile, g);
#pragma unroll
        for (int w = QT - 1; w >= 0; --w)   // small terms first
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][tile] = mma(k, q[rt][g][w], s[rt][tile]);
      }
    }
  }
  // what a row does not see of the block from t0 on; window: tokens up to its last one that it sees (0: all)
  __device__ __forceinline__ void mask(f32x4 (&s)[RT][2], int t0, int quarter, int window) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int low = window > 0 ? last[rt] - window : -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int t = t0 + (e >> 2) * 16 + quarter * 4 + (e & 3);
        s[rt][e >> 2][e & 3] = t <= last[rt] && t > low ? s[rt][e >> 2][e & 3] : -INFINITY;
      }
    }
  }
  // raises the running maximum of tile rt where a score passes it by a factor of more than 2^8
  __device__ __forceinline__ void raise(const f32x4 (&s)[2], int rt, float scale_log2) {
    float hi = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
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
  }
  // 2^(score - maximum) as PT terms, and their sum: scores 2 i and 2 i + 1 of a lane's eight
  __device__ __forceinline__ void weigh(const f32x4 (&s)[2], int rt, int i, float scale_log2, Frag (&p)[PT]) {
    const float ref = top[rt] == -INFINITY ? 0.f : top[rt];
    float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][2 * (i & 1)], scale_log2, -ref));
    float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][2 * (i & 1) + 1], scale_log2, -ref));
    sum[rt] += x + y;
#pragma unroll
    for (int w = 0; w < PT; ++w) p[w].u[i] = take_pair(x, y, w + 1 < PT);
  }
  __device__ __forceinline__ void add_values(int g, const Frag& even, const Frag& odd, const Frag (&p)[RT][PT]) {
#pragma unroll
    for (int w = PT - 1; w >= 0; --w)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        acc[rt][2 * g] = mma(even, p[rt][w], acc[rt][2 * g]);
        acc[rt][2 * g + 1] = mma(odd, p[rt][w], acc[rt][2 * g + 1]);
      }
  }
  // plain: every row sees all 32 tokens (uniform).  The masks are behind a branch that holds an empty asm volatile: without it the compiler
  // makes selects of them, for every block.
  __device__ __forceinline__ void step(const BlockBytes<M>& b, int t0, int len, bool plain, float scale_log2, int quarter, int window) {
    f32x4 s[RT][2];
    scores(b, s);
    uint32_t keep[2] = {~0u, ~0u};   // bytes of the tokens that exist, of this lane's 4 + 4
    if (!plain) {
      asm volatile("" ::: );
      keep_of(keep, len - t0, quarter);
      mask(s, t0, quarter, window);
    }
    Frag p[RT][PT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      raise(s[rt], rt, scale_log2);
#pragma unroll
      for (int i = 0; i < 4; ++i) weigh(s[rt], rt, i, scale_log2, p[rt]);
    }
#pragma unroll
    for (int g = 0; g < M; ++g) {
      Frag even, odd;
      b.values(g, plain, keep, even, odd);
      add_values(g, even, odd, p);
    }
  }
};

// eight elements of an output row from d0 on, relative to the maximum `top`
template <int M, Elem E>
__device__ __forceinline__ void put_row(const Kv4Attention& a, int split, int64_t row, int h, int d0, const float* v, float top, float sum, bool first) {
  typedef typename ElemOf<E>::T T;
  constexpr int DP = 32 * M;
  if (a.nsplit > 1) {
    float* p = a.part + ((row * a.heads + h) * a.nsplit + split) * (DP + kPartPad);
    *reinterpret_cast<float4*>(p + d0) = float4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4*>(p + d0 + 4) = float4{v[4], v[5], v[6], v[7]};
    if (first) p[DP] = top, p[DP + 1] = sum;
    return;
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
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
  if (first && a.lse != nullptr) a.lse[row * a.heads + h] = sum != 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f : -INFINITY;
}

// a wave's own rows
template <int M, Elem E, int RT>
__device__ __forceinline__ void put_walk(const Kv4Attention& a, int split, const Walk<M, E, RT>& w, int row0, int n_rows, int64_t q0, int head, int per, int lane) {
  const int quarter = lane >> 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + (lane & 15), tq = r / per;
    if (r >= n_rows) continue;
#pragma unroll
    for (int g = 0; g < M; ++g) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[2 * r] = w.acc[rt][2 * g][r], v[2 * r + 1] = w.acc[rt][2 * g + 1][r];
      put_row<M, E>(a, split, q0 + tq, head * per + r - tq * per, g * 32 + quarter * 8, v, w.top[rt], w.sum[rt], g == 0 && quarter == 0);
    }
  }
}

// KW: waves that share 16 * RT rows, take the blocks of the workgroup's range in turn and join their results in shared memory; 4 / KW such
//   units (a tile of rows of a sequence and key / value head) make a workgroup.
// waves per SIMD: left alone the compiler spends the registers of two or three waves on one; asked for more it spills
template <int M, Elem E, int RT>
constexpr int waves_wanted() {
  if (RT == 1) return kv4_attention_waves(M, E == Elem::f32);
  return M <= 2 ? (E == Elem::bf16 ? 3 : 2) : M <= 4 ? 2 : 1;
}
template <int M, Elem E, int RT, int KW>
__global__ __launch_bounds__(256, (waves_wanted<M, E, RT>())) void kv4_attention_kernel(Kv4Attention a) {
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
  w.begin(a, row0, n_rows, n_q, len, active ? q0 : 0, head, per, quarter, idx);

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
  // 64 entries of the table at a time, one a lane: a load of each would be waited for in every turn
  const int last_page = (blk1 - 1) >> in_shift;
  int held = blk0 >> in_shift;
  int32_t entries = blk0 < blk1 ? table[min(held + lane, last_page)] : -1;
  // (blocks behind the last are the last again, and a page that is not in the cache is page 0, not looked at: the loads of a step are
  // unconditional, or each would be waited for where its condition ends)
  auto page_of = [&](int blk) -> int32_t {
    const int i = min(blk, blk1 - 1) >> in_shift;
    if (i - held >= 64) held = i, entries = table[min(held + lane, last_page)];
    return __builtin_amdgcn_readlane(entries, i - held);
  };
  const uint32_t pages = a.cache.pages < INT_MAX ? (uint32_t)a.cache.pages : (uint32_t)INT_MAX;
  auto good = [&](int32_t page) { return (uint32_t)page < pages; };
  auto at = [&](int blk, int32_t page) {
    return a.cache.data + ((((int64_t)(good(page) ? page : 0) * heads_kv + head) << in_shift) + ((blk < blk1 ? blk : blk1 - 1) & in_mask)) * block_bytes;
  };
  auto plain = [&](int blk) { return blk * 32 >= all_from && blk * 32 + 32 <= all_to && blk * 32 + 32 <= len; };

  constexpr int step = KW;
  int blk = blk0 + sub;
  if (blk < blk1) {
    BlockBytes<M> x, y;
    int32_t px = page_of(blk), py = page_of(blk + step);
    auto walk = [&](const BlockBytes<M>& bytes) { w.step(bytes, blk * 32, len, plain(blk), a.scale_log2, quarter, a.window); };
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

  auto finish = [&](int64_t row, int h, int d0, const float* v, float top, float sum, bool first) { put_row<M, E>(a, split, row, h, d0, v, top, sum, first); };

  if constexpr (KW == 1) {
    put_walk<M, E, RT>(a, split, w, row0, n_rows, q0, head, per, lane);
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

// ---- chunks of prompts --------------------------------------------------------------------------------------------------
// The same walk for many rows: a workgroup has 64 * RT rows, a wave 16 * RT of them, and all four walk the same blocks.  The matrix operands of
// a block are expanded ONCE, a quarter by each wave, into shared memory (in the order in which a wave reads them back: 16 bytes a lane, no
// conflicts), two blocks deep: one barrier a block, the bytes of later blocks in flight meanwhile.
// 4 sequences of 2500 to 8191 tokens with 485 to 1000 queries, 32 over 8 heads of 128, f16: 550 us and 36 for the join, 490 TFLOP/s of the formula's
// products.  Two terms of q and of p make each of them two on the matrix unit, which is busy half of the time and the vector unit (softmax, terms, expanding)
// the other half, at 2.1 GHz: what is left is their overlap.  Each wave expanding for itself: 740 us; operands read where they are used: 720.  bf16, one term
// of q: 467 and 34 us; fp32, three of each: 861 and 34.
// a wave's quarter of a block: keys' operands wave, wave + 4, ... of 2 M and values' groups (wave + 2) % 4, + 4, ... of M
template <int M>
struct QuarterKeys {
  static constexpr int N = (2 * M + 3) / 4;
  uint32_t k[N], s[N];

  __device__ __forceinline__ void load(const uint8_t* b, int wave, int lane) {
    const int quarter = lane >> 4, idx = lane & 15;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int f = min(wave + 4 * i, 2 * M - 1), tile = f / M, g = f - tile * M;
      k[i] = *reinterpret_cast<const uint32_t*>(b + (uint32_t)kv4_key_at(tile * 16 + idx, g, quarter, M));
      s[i] = b[(uint32_t)kv4_key_scale_at(tile * 16 + idx, g, M)];
    }
  }
  __device__ __forceinline__ void expand(Frag* f, int wave, int i) const {
    if (4 * i + 4 <= 2 * M || wave + 4 * i < 2 * M) f[(wave + 4 * i) * 64] = expand_keys(k[i], s[i], 0);
  }
};
template <int M>
struct QuarterValues {
  static constexpr int N = (M + 3) / 4;
  uint2 v[N], s[N];

  __device__ __forceinline__ void load(const uint8_t* b, int wave, int lane) {
    const int quarter = lane >> 4, idx = lane & 15;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = min(((wave + 2) & 3) + 4 * i, M - 1);
      v[i] = *reinterpret_cast<const uint2*>(b + (uint32_t)kv4_value_at(quarter * 4, g, idx, M));
      s[i] = *reinterpret_cast<const uint2*>(b + (uint32_t)kv4_value_scale_at(quarter * 4, g, M));
    }
  }
  __device__ __forceinline__ void expand(Frag* f, int wave, const uint32_t* keep, int i) const {
    const int g = ((wave + 2) & 3) + 4 * i;
    if (4 * i + 4 > M && g >= M) return;
    const uint32_t codes[2] = {v[i].x, v[i].y}, scales[2] = {keep_scales(s[i].x, keep[0]), keep_scales(s[i].y, keep[1])};
    Frag even, odd;
    expand_values(codes, scales, even, odd);
    f[2 * g * 64] = even;
    f[(2 * g + 1) * 64] = odd;
  }
};

template <int M, Elem E, int RT>
__global__ __attribute__((amdgpu_waves_per_eu((M <= 4 ? 2 : 1), (M <= 4 ? 2 : 1)))) __launch_bounds__(256) void kv4_attention_chunk_kernel(Kv4Attention a) {
  __shared__ Frag keys[2][2 * M][64], values[2][2 * M][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int quarter = lane >> 4, idx = lane & 15;
  const int heads_kv = a.cache.heads, per = a.heads / heads_kv;
  // workgroups go round the eight XCDs: pair p = (sequence, key / value head) belongs to XCD p % 8, so that the tiles that read one head's
  // pages share an L2, and every XCD has heads of every sequence.  A number of pairs that is not a multiple of eight leaves XCDs idle: 1, 2, 3, 4 or 5 pairs
  // take as long as 8 (2.3 ms, 4160 queries of 16 heads each over 8192 tokens of one head of 128, bf16), 9 as long as 16 (4.5 ms)
  const int turn = (int)blockIdx.x >> 3, unit = turn / a.nsplit, split = turn - unit * a.nsplit;
  const int group = unit / a.tiles, pair = group * 8 + ((int)blockIdx.x & 7), tile0 = unit - group * a.tiles;
  const int b = pair / heads_kv, head = pair - b * heads_kv, page_shift = a.cache.page_shift;
  if (b >= a.batch) return;
  const int64_t q0 = a.q_start != nullptr ? a.q_start[b] : (int64_t)b * a.max_q;
  int n_q = a.q_start != nullptr ? a.q_start[b + 1] - a.q_start[b] : a.max_q;
  if (n_q > a.max_q) n_q = a.max_q;
  if (q0 < 0 || n_q <= 0 || q0 + n_q > a.rows) return;   // (a q_start that does not fit: nothing is written)
  const int n_rows = n_q * per, first_row = tile0 * 64 * RT;
  if (first_row >= n_rows) return;
  int len = a.kv_lens[b];
  const int64_t room = (int64_t)a.width << page_shift;
  len = len < 0 ? 0 : len > room ? (int)room : len;

  const int row0 = first_row + wave * 16 * RT;
  Walk<M, E, RT> w;
  w.begin(a, row0, n_rows, n_q, len, q0, head, per, quarter, idx);
  // tokens that some / every row from r0 to r1 sees
  struct Span {
    int from, to, all_from, all_to;
  };
  auto span_of = [&](int r0, int r1) {
    const int t0 = r0 / per, t1 = r1 / per, base = len - n_q;
    Span s{0, len, 0, len};
    if (a.causal) {
      s.to = max(base + t1 + 1, 0), s.all_to = base + t0 + 1;
      if (a.window > 0) s.from = max(base + t0 - a.window + 1, 0), s.all_from = base + t1 - a.window + 1;
    }
    return s;
  };
  const Span all = span_of(first_row, min(first_row + 64 * RT, n_rows) - 1);
  Span own = span_of(min(row0, n_rows - 1), min(row0 + 16 * RT, n_rows) - 1);
  if (row0 >= n_rows) own.to = 0;
  int blk0 = all.from >> 5, blk1 = (all.to + 31) >> 5;
  if (a.nsplit > 1) {
    const int share = (blk1 - blk0 + a.nsplit - 1) / a.nsplit;
    blk0 += split * share;
    blk1 = min(blk0 + share, blk1);
  }
  const int32_t* table = a.table + (int64_t)b * a.width;
  const int64_t block_bytes = kv4_block_bytes(M);
  const int in_shift = page_shift - 5, in_mask = (1 << in_shift) - 1;
  // 64 entries of the table at a time, one a lane
  int held = blk0 >> in_shift;
  const int last_page = (blk1 - 1) >> in_shift;
  int32_t entries = blk0 < blk1 ? table[min(held + lane, last_page)] : -1;
  auto page_of = [&](int blk) -> int32_t {
    const int i = min(blk, blk1 - 1) >> in_shift;
    if (i - held >= 64) held = i, entries = table[min(held + lane, last_page)];
    return __builtin_amdgcn_readlane(entries, i - held);
  };
  const uint32_t pages = a.cache.pages < INT_MAX ? (uint32_t)a.cache.pages : (uint32_t)INT_MAX;
  auto good = [&](int32_t page) { return (uint32_t)page < pages; };
  auto at = [&](int blk, int32_t page) {   // (a page that is not in the cache: page 0, not looked at)
    return a.cache.data + ((((int64_t)(good(page) ? page : 0) * heads_kv + head) << in_shift) + (min(blk, blk1 - 1) & in_mask)) * block_bytes;
  };
  if (blk0 < blk1) {
    // Turn of block n: scores of block n + 1 beside the softmax of block n (one needs the matrix unit, the other the vector unit), then
    // block n's values; keys of block n + 2 and values of block n + 1 are expanded meanwhile, and their successors' bytes loaded.  The
    // barriers to the compiler's scheduling keep it that way: left alone it reads an operand right before its product and waits.
    typedef Walk<M, E, RT> W;
    QuarterKeys<M> rk;
    QuarterValues<M> rv;
    int32_t page[4] = {page_of(blk0), page_of(blk0 + 1), page_of(blk0 + 2), page_of(blk0 + 3)};
    f32x4 s[2][RT][2];
    // products [from, to) of a block's scores, in the order group, term (small ones first), token tile, row tile
    constexpr int kPer = 2 * RT * W::QT, kProducts = M * kPer;
    Frag kf[2][2];
    auto read_keys = [&](const Frag* k, int g) { kf[g & 1][0] = k[g * 64], kf[g & 1][1] = k[(M + g) * 64]; };
    auto products = [&](const Frag* k, f32x4 (&out)[RT][2], int from, int to) {
#pragma unroll
      for (int m = 0; m < kProducts; ++m) {
        if (m < from || m >= to) continue;
        const int g = m / kPer, in = m % kPer, t = W::QT - 1 - in / (2 * RT), tile = in / RT % 2, rt = in % RT;
        if (in == 0 && g + 1 < M) read_keys(k, g + 1);
        out[rt][tile] = mma(kf[g & 1][tile], w.q[rt][g][t], m < 2 * RT ? f32x4{0.f, 0.f, 0.f, 0.f} : out[rt][tile]);
      }
    };
    uint32_t keep[2];
    rk.load(at(blk0, page[0]), wave, lane);
    rv.load(at(blk0, page[0]), wave, lane);
#pragma unroll
    for (int i = 0; i < rk.N; ++i) rk.expand(&keys[0][0][lane], wave, i);
    keep_of(keep, len - blk0 * 32, quarter);
#pragma unroll
    for (int i = 0; i < rv.N; ++i) rv.expand(&values[0][0][lane], wave, keep, i);
    rk.load(at(blk0 + 1, page[1]), wave, lane);
    rv.load(at(blk0 + 1, page[1]), wave, lane);
#pragma unroll
    for (int i = 0; i < rk.N; ++i) rk.expand(&keys[1][0][lane], wave, i);
    rk.load(at(blk0 + 2, page[2]), wave, lane);
    __syncthreads();
    read_keys(&keys[0][0][lane], 0);
    products(&keys[0][0][lane], s[0], 0, kProducts);
    __syncthreads();
    auto turn = [&](int blk, int cur) {
      const int32_t after = page_of(blk + 4);
      const int t0 = blk * 32;
      const Frag *k = &keys[cur ^ 1][0][lane], *v = &values[cur][0][lane];
      constexpr int kPieces = rk.N + rv.N;
      auto expand = [&](int i) {
        if (i < rk.N) rk.expand(&keys[cur][0][lane], wave, i);
        else rv.expand(&values[cur ^ 1][0][lane], wave, keep, i - rk.N);
      };
      read_keys(k, 0);
      keep[0] = keep[1] = ~0u;
      if (t0 + 64 > len) {
        asm volatile("" ::: );
        keep_of(keep, len - t0 - 32, quarter);
      }
      if (good(page[0]) && t0 < own.to && t0 + 32 > own.from) {
        if (t0 < own.all_from || t0 + 32 > own.all_to || t0 + 32 > len) {
          asm volatile("" ::: );
          w.mask(s[cur], t0, quarter, a.window);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) w.raise(s[cur][rt], rt, a.scale_log2);
        Frag p[RT][W::PT], vf[2][2];
        constexpr int kSlices = 4 * RT;
#pragma unroll
        for (int i = 0; i < kSlices; ++i) {
          products(k, s[cur ^ 1], kProducts * i / kSlices, kProducts * (i + 1) / kSlices);
          w.weigh(s[cur][i >> 2], i >> 2, i & 3, a.scale_log2, p[i >> 2]);
          if (i == kSlices - 2) vf[0][0] = v[0], vf[0][1] = v[64];
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int g = 0; g < M; ++g) {
          if (g + 1 < M) vf[(g + 1) & 1][0] = v[2 * (g + 1) * 64], vf[(g + 1) & 1][1] = v[(2 * g + 3) * 64];
#pragma unroll
          for (int i = 0; i < kPieces; ++i)
            if ((i < M - 1 ? i : M - 1) == g) expand(i);
          w.add_values(g, vf[g & 1][0], vf[g & 1][1], p);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        products(k, s[cur ^ 1], 0, kProducts);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) expand(i);
      }
      rk.load(at(blk + 3, page[3]), wave, lane);
      rv.load(at(blk + 2, page[2]), wave, lane);
      page[0] = page[1], page[1] = page[2], page[2] = page[3], page[3] = after;
      __syncthreads();
    };
    for (int blk = blk0; blk < blk1; blk += 2) {
      turn(blk, 0);
      if (blk + 1 < blk1) turn(blk + 1, 1);
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    w.sum[rt] += __shfl_xor(w.sum[rt], 16);
    w.sum[rt] += __shfl_xor(w.sum[rt], 32);
  }
  put_walk<M, E, RT>(a, split, w, row0, n_rows, q0, head, per, lane);
}

// Joins the key ranges of one (row, head): one wave each, or the WAVES = 4 of a workgroup where rows are few and ranges many.  What it waits for is loads, so
// all are on their way before the first is used, the row's owner looked up meanwhile.  96 rows of 256, 26 ranges: 5.4 us by four waves, 10.4 by one; 512 rows of
// 128, 15 ranges: 4.8 and 5.1; 95040 rows of 128, two ranges, one wave each: 36 us, 3.4 TB/s.
// kFirst: turns whose loads do not wait for anything (one where one is all there is)
template <Elem E, int kFirst, int WAVES>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4Attention a, int dp) {
  typedef typename ElemOf<E>::T T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = WAVES > 1 ? wave : 0;
  const uint32_t id = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const uint32_t row = id / (uint32_t)a.heads;
  const int h = (int)(id - row * a.heads);
  if (row >= a.rows) return;
  // lane s: the maximum and the sum of range s (at most 64 of them)
  const int64_t stride = dp + kPartPad;
  const float* p = a.part + ((int64_t)row * a.heads + h) * a.nsplit * stride;
  const float2 stat = *reinterpret_cast<const float2*>(p + min(lane, a.nsplit - 1) * stride + dp);
  // a lane has four elements; where those take up half the wave or less, groups of lanes take the ranges in turn.  (Every lane takes every turn:
  // the shuffles read lanes of all groups.)
  const int per = dp >> 2, groups = 64 / per, group = lane / per, d0 = (lane - group * per) * 4;
  const bool has = group < groups;
  auto range = [&](int turn) { return (turn * groups + (has ? group : 0)) * WAVES + part; };
  auto piece = [&](int turn) { return *reinterpret_cast<const float4*>(p + min(range(turn), a.nsplit - 1) * stride + d0); };
  float4 first[kFirst];
#pragma unroll
  for (int i = 0; i < kFirst; ++i) first[i] = piece(i);
  // rows that no sequence owns are left as they are
  bool owned = true;
  if (a.q_start != nullptr) {
    int lo = 0, hi = a.batch;
    while (lo < hi) {   // last sequence that starts at or before the row
      const int mid = (lo + hi + 1) >> 1;
      if (mid < a.batch && a.q_start[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    const int64_t q0 = a.q_start[lo], q1 = a.q_start[lo + 1];
    owned = row >= q0 && row < q1 && row < q0 + a.max_q && q0 >= 0 && (q1 - q0 > a.max_q ? q0 + a.max_q : q1) <= a.rows;
  }
  if (!owned) return;
  const float mine = lane < a.nsplit ? stat.x : -INFINITY;
  float top = mine;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - top);
  float sum = lane < a.nsplit ? stat.y * f : 0.f;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  float4 v{0.f, 0.f, 0.f, 0.f};
  auto add = [&](int turn, const float4& x) {
    const int s = range(turn);
    const float g = __shfl(f, s & 63);
    if (s < a.nsplit && has) v.x += x.x * g, v.y += x.y * g, v.z += x.z * g, v.w += x.w * g;
  };
  const int turns = (a.nsplit + groups * WAVES - 1) / (groups * WAVES);
#pragma unroll
  for (int i = 0; i < kFirst; ++i) add(i, first[i]);
  if (kFirst > 1) {
#pragma unroll 8
    for (int i = kFirst; i < turns; ++i) add(i, piece(i));
  }
  for (int k = 1; k < groups; ++k) {
    const float4 x{__shfl(v.x, lane + k * per), __shfl(v.y, lane + k * per), __shfl(v.z, lane + k * per), __shfl(v.w, lane + k * per)};
    if (group == 0) v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
  }
  if constexpr (WAVES > 1) {
    __shared__ float4 sums[WAVES][64];
    sums[wave][lane] = v;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 x = sums[w][lane];
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
  }
  if (group == 0) {
    T* o = static_cast<T*>(a.out) + (int64_t)row * a.out_row + h * a.out_head;
    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    if (a.fm == nullptr && a.vec) {
      if (d0 < a.cache.head_dim) store_elems<E, 4>(o + d0, y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = d0 + e;
        if (d >= a.cache.head_dim) break;
        if (a.fm != nullptr) a.fm[fm16((int)row, h * a.cache.head_dim + d, a.heads * a.cache.head_dim >> 5)] = ElemOf<Elem::bf16>::put(y[e]);
        else o[d] = ElemOf<E>::put(y[e]);
      }
    }
  }
  if (lane == 0 && a.lse != nullptr) a.lse[(int64_t)row * a.heads + h] = sum != 0.f ? (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f : -INFINITY;
}

template <int M, Elem E>
void launch_kv4_attention(const Kv4Attention& a0, hipStream_t s) {
  Kv4Attention a = a0;
  const Kv4Shape shape = kv4_attention_shape(a, E);
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads);
  a.tiles = (int32_t)((rows + shape.rows() - 1) / shape.rows());
  const int64_t four = E == Elem::f32 ? 16 : 8;   // bytes of four elements
  const int64_t size = four / 4;
  auto even = [&](const void* p, int64_t row, int64_t head) { return (uintptr_t)p % four == 0 && row * size % four == 0 && head * size % four == 0; };
  a.vec = a.cache.head_dim % 4 == 0 && even(a.q, a.q_row, a.q_head) && (a.fm != nullptr || even(a.out, a.out_row, a.out_head));
  a.window = a.window < (1 << 30) ? a.window : 1 << 30;   // (no table has more tokens, and places minus this stay in 32 bits)
  a.sign = a.scale_log2 < 0.f ? -1.f : 1.f;
  a.scale_log2 = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);   // (0 * -inf of a masked score would be NaN; any score times this is 0 to exp2)
  if (shape.chunk) {
    const dim3 grid((unsigned)kv4_attention_groups(a, E));
    MSH_LAUNCH((kv4_attention_chunk_kernel<M, E, 2>), grid, dim3(256), 0, s, a);
  } else {
    const dim3 grid((unsigned)kv4_attention_groups(a, E), (unsigned)a.nsplit);
    if (shape.rt == 1 && shape.kw == 4) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 4>), grid, dim3(256), 0, s, a);
    else if (shape.rt == 1 && shape.kw == 2) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 2>), grid, dim3(256), 0, s, a);
    else if (shape.rt == 1) MSH_LAUNCH((kv4_attention_kernel<M, E, 1, 1>), grid, dim3(256), 0, s, a);
    else if constexpr (M <= 2 || E != Elem::f32) MSH_LAUNCH((kv4_attention_kernel<M, E, 2, 4>), grid, dim3(256), 0, s, a);   // (kv4_attention_shape())
  }
  if (a.nsplit == 1) return;
  const int64_t joins = a.rows * a.heads;
  const dim3 by_wave((unsigned)kv4_join_groups(a.rows, a.heads)), by_group((unsigned)joins);
  constexpr int groups = 64 / (8 * M);   // ranges that a wave takes at a time
  if (a.nsplit > 2 * groups && joins <= 1024) MSH_LAUNCH((kv4_join_kernel<E, 4, 4>), by_group, dim3(256), 0, s, a, 32 * M);
  else if (a.nsplit > groups) MSH_LAUNCH((kv4_join_kernel<E, 4, 1>), by_wave, dim3(256), 0, s, a, 32 * M);
  else MSH_LAUNCH((kv4_join_kernel<E, 1, 1>), by_wave, dim3(256), 0, s, a, 32 * M);
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
