// The paged 4-bit cache: plan of pages and slots, writing rows, reading rows (form: serve_kernels.h).
#include "kv4_common.h"

namespace msh {
namespace {

// ---- plan ---------------------------------------------------------------------------------------------------------------
// need_b = ceil(len_b / P), kept_b = ceil((len_b - new_b) / P), first_b = sum of need - kept over the requests before b; table entry
// kept_b + i of request b becomes free[first_b + i], and the row at place p of request b the slot table[b][p / P] * P + p mod P.
// One launch, one workgroup per request: each adds up the lengths of the requests before it for itself (8 bytes each, out of L2) instead of
// waiting for a scan of its own launch, and clears the rows between its own and the next request's.  A few bytes per request: bound by
// launch and memory latency.  5 requests 2.9 us, 1999 with up to 16000 tokens each 6.1 us.  (The sums grow with the square of the requests: a plan of tens of
// thousands would want a scan.)
struct Plan {
  int32_t* table;
  const int32_t *kv_lens, *new_lens, *row_start, *free_pages;
  int64_t* slots;
  int32_t* used;
  int64_t rows, n_free;
  int32_t batch, width, page_shift;
};

__device__ __forceinline__ void plan_lens(const Plan& p, int b, int& held, int& fresh) {
  const int most = p.width << p.page_shift;   // (at most 2^30)
  held = p.kv_lens[b], fresh = p.new_lens[b];
  held = held < 0 ? 0 : held > most ? most : held;
  fresh = fresh < 0 ? 0 : fresh > held ? held : fresh;
}
__device__ __forceinline__ int pages_of(int tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

__global__ __launch_bounds__(256) void page_plan_kernel(Plan p) {
  __shared__ int64_t red[4];
  const int b = blockIdx.x, shift = p.page_shift;
  int held, fresh;
  plan_lens(p, b, held, fresh);
  const int64_t start = p.row_start[b], next = b + 1 < p.batch ? p.row_start[b + 1] : p.rows;
  int64_t first = 0;   // pages taken by the requests before b
  for (int i = threadIdx.x; i < b; i += 256) {
    int h, f;
    plan_lens(p, i, h, f);
    first += pages_of(h, shift) - pages_of(h - f, shift);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) first += __shfl_xor(first, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = first;
  __syncthreads();
  first = red[0] + red[1] + red[2] + red[3];
  const int kept = pages_of(held - fresh, shift), need = pages_of(held, shift);
  if (b == p.batch - 1 && threadIdx.x == 0) *p.used = (int32_t)min(first + need - kept, (int64_t)INT_MAX);
  int32_t* row = p.table + (int64_t)b * p.width;
  auto page_at = [&](int c) -> int32_t {   // (kept entries are read, the others written: by no other workgroup)
    if (c < kept) return row[c];
    const int64_t at = first + c - kept;
    return c < need && at < p.n_free ? p.free_pages[at] : -1;
  };
  const int64_t from = b == 0 ? 0 : start, to = next < p.rows ? next : p.rows;   // rows this request answers for
  for (int64_t at = from + threadIdx.x; at < to; at += 256) {
    int64_t slot = -1;
    const int64_t i = at - start;
    if (i >= 0 && i < fresh) {
      const int place = held - fresh + (int)i;
      const int32_t page = page_at(place >> shift);
      if (page >= 0) slot = ((int64_t)page << shift) + (place & ((1 << shift) - 1));
    }
    if (at >= 0) p.slots[at] = slot;
  }
  for (int c = kept + threadIdx.x; c < p.width; c += 256) row[c] = page_at(c);
}

// ---- writing ------------------------------------------------------------------------------------------------------------
// e = floor(log2(amax)) - 2, one more where the mantissa is 1.75 or above: amax / 2^e lies in [3.5, 7), and what saturates at 6 or
// rounds at 3.5 is off by a seventh at most.  NaN is stored as 0, infinities as the largest finite value.
__device__ __forceinline__ float storable(float x) {
  x = x != x ? 0.f : x;
  return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
}
// the largest magnitude's bits, which are ordered as the magnitudes are (infinity and NaN above all)
__device__ __forceinline__ uint32_t abs_max8(const float* x) {
  uint32_t a = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(x[e]) & 0x7fffffffu);
  return a;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)((amax_bits + 0x200000u) >> 23) - 129;
  return (uint32_t)((e < -100 ? -100 : e > 125 ? 125 : e) + 127);
}
__device__ __forceinline__ uint32_t codes8(const float* x, float scale) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
  return r;
}

// A workgroup: 4 rows x 16 (head, group) pairs x 4 quarters, a thread 8 elements of a key and of a value; its reads of a row are contiguous
// over the heads.  Where four neighbouring rows are the four tokens of one aligned run of slots -- every prompt -- their lanes
// exchange the value bytes (16 neighbouring lanes hold 4 tokens x 4 quarters) and store one dword of four tokens each instead of four
// bytes.  One (head, group) a thread: a loop over the groups measured slower (its loads wait for one another).
// 53120 bf16 rows of 8 heads of 52 (117 MB): 28 us, 4.2 TB/s, by the vector unit (scales, codes, the exchange; with floats made of the 16-bit elements
// first it was 33) beside HBM; reading them back 24 us, 4.9 TB/s, what a copy reaches.  61 rows of 8 heads of 128: 3.5 us each, a launch.
__device__ __forceinline__ uint32_t lanes_rotate4(uint32_t x) {   // from the lane 4 below within the 16, cyclically
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x124 /* row_ror:4 */, 0xf, 0xf, false);
}
// lane c (of four lanes 4 apart) holds bytes [i] of token c; returns bytes [token] of pair i = c
__device__ __forceinline__ uint32_t transpose4(uint32_t x, int c) {
  uint32_t out = ((x >> (8 * c)) & 255u) << (8 * c);
#pragma unroll
  for (int s = 1; s < 4; ++s) {
    x = lanes_rotate4(x);
    const int from = (c - s) & 3;   // the token the word came from
    out |= ((x >> (8 * c)) & 255u) << (8 * from);
  }
  return out;
}

struct Item {      // of a thread
  int64_t r, slot;
  int h, g, quarter, tok;
  bool live, four;   // four: this lane's four rows are the four tokens of an aligned run
};
template <int m>
__device__ __forceinline__ Item item_of(const Kv4Cache& c, const int64_t* slots, int64_t rows) {
  Item it;
  it.quarter = threadIdx.x & 3, it.tok = (threadIdx.x >> 2) & 3;
  const int pair = (int)blockIdx.y * 16 + (threadIdx.x >> 4);
  it.h = pair / m, it.g = pair - it.h * m;
  // workgroups go round the eight XCDs: each takes a contiguous eighth of the rows, so that the eight workgroups that share a block's
  // lines share an L2 (gridDim.x is a multiple of eight)
  const uint32_t eighth = gridDim.x >> 3;
  it.r = (int64_t)((blockIdx.x & 7) * eighth + (blockIdx.x >> 3)) * 4 + it.tok;
  const bool in = it.r < rows && it.h < c.heads;
  it.slot = in ? slots[it.r] : -1;
  it.live = it.slot >= 0 && it.slot < c.pages << c.page_shift;
  return it;
}
// (kept apart: the element loads are issued before the slot is looked at)
__device__ __forceinline__ void item_run(Item& it) {
  const uint32_t run = it.live ? (uint32_t)(it.slot >> 2) : 0u, run_hi = it.live ? (uint32_t)(it.slot >> 34) : 0u;
  uint32_t a = run, b = run_hi, ok = it.live && (int)(it.slot & 3) == it.tok ? 1u : 0u, all = ok;
#pragma unroll
  for (int s = 1; s < 4; ++s) {
    a = lanes_rotate4(a), b = lanes_rotate4(b), ok = lanes_rotate4(ok);
    all &= ok & (a == run && b == run_hi ? 1u : 0u);
  }
  // (live, the same run and each its own place: that is the same answer in all four lanes)
  it.four = all != 0;
}
__device__ __forceinline__ uint8_t* item_block(const Kv4Cache& c, const Item& it, int m, int& t) {
  const int64_t page = it.slot >> c.page_shift;
  const int place = (int)(it.slot & ((1 << c.page_shift) - 1));
  t = place & 31;
  return c.data + (((page * c.heads + it.h) << (c.page_shift - 5)) + (place >> 5)) * kv4_block_bytes(m);
}

// eight elements of a thread as they are read: floats, or 16-bit elements in pairs, whose largest magnitude and codes take half the instructions
template <Elem E>
struct Eight {
  uint32_t w[4];
  __device__ __forceinline__ void load4(const void* p, int half) {
    const uint2 u = *static_cast<const uint2*>(p);
    w[2 * half] = u.x, w[2 * half + 1] = u.y;
  }
  __device__ __forceinline__ void set(int e, uint16_t v) { w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | (uint32_t)v << 16 : v; }
  __device__ __forceinline__ void clear_from(int n) {   // elements n and behind (n a constant after unrolling, or the row's end)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i >= n ? 0u : 2 * i + 1 >= n ? w[i] & 0xffffu : w[i];
  }
  __device__ __forceinline__ uint32_t abs_max() const {   // as the bits of a float
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    const uint32_t a = max((uint32_t)m[0], (uint32_t)m[1]);
    if constexpr (E == Elem::bf16) return a << 16;
    return __float_as_uint(ElemOf<E>::get((typename ElemOf<E>::T)a));
  }
  __device__ __forceinline__ void floats(float* x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t v = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      x[e] = ElemOf<E>::get((typename ElemOf<E>::T)v);
    }
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t r = 0;
    if constexpr (E == Elem::bf16) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
    } else {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w[0]), scale, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w[1]), scale, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w[2]), scale, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w[3]), scale, 3);
    }
    return r;
  }
};
template <>
struct Eight<Elem::f32> {
  float x[8];
  __device__ __forceinline__ void load4(const void* p, int half) { load_elems<Elem::f32, 4>(static_cast<const float*>(p), x + 4 * half); }
  __device__ __forceinline__ void set(int e, float v) { x[e] = v; }
  __device__ __forceinline__ void clear_from(int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e >= n ? 0.f : x[e];
  }
  __device__ __forceinline__ uint32_t abs_max() const { return abs_max8(x); }
  __device__ __forceinline__ void floats(float* y) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e];
  }
  __device__ __forceinline__ uint32_t codes(float scale) const { return codes8(x, scale); }
};

template <Elem E, int M>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4Cache c, Kv4Rows k, Kv4Rows v, int64_t rows, const int64_t* slots, int vec) {
  typedef typename ElemOf<E>::T T;
  constexpr int m = M;   // (groups of 32: the offsets below become shifts and adds)
  Item it = item_of<M>(c, slots, rows);
  const int g = it.g, quarter = it.quarter, d0 = g * 32 + quarter * 8;
  const bool in = it.r < rows && it.h < c.heads;
  const T* kp = static_cast<const T*>(k.p) + it.r * k.row + it.h * k.head;
  const T* vp = static_cast<const T*>(v.p) + it.r * v.row + it.h * v.head;
  Eight<E> x[2];
  x[0].clear_from(0), x[1].clear_from(0);
  // (loads are clamped into the row and selected afterwards: none waits for another)
  if (in && vec) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int d = d0 + e + 4 <= c.head_dim ? d0 + e : c.head_dim - 4;
      x[0].load4(kp + d, e >> 2);
      x[1].load4(vp + d, e >> 2);
    }
  } else if (in) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e < c.head_dim ? d0 + e : c.head_dim - 1;
      x[0].set(e, kp[d * k.elem]);
      x[1].set(e, vp[d * v.elem]);
    }
  }
  x[0].clear_from(c.head_dim - d0), x[1].clear_from(c.head_dim - d0);
  item_run(it);
  uint32_t codes[2], scale[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t own = x[w].abs_max();
    uint32_t a = own;
    float y[8];
    if (own >= 0x7f800000u) {   // an infinity or NaN: rare
      x[w].floats(y);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = storable(y[e]);
      a = abs_max8(y);
    }
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1 /* quad_perm 1,0,3,2 */, 0xf, 0xf, false));
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E /* quad_perm 2,3,0,1 */, 0xf, 0xf, false));
    scale[w] = scale_byte(a);
    codes[w] = x[w].codes(kv4_scale(scale[w]));
    if (own >= 0x7f800000u) codes[w] = codes8(y, kv4_scale(scale[w]));
  }
  const uint32_t run = transpose4(codes[1], it.tok);   // (every lane takes part in the exchange)
  if (!it.live) return;
  int t;
  uint8_t* b = item_block(c, it, m, t);
  *reinterpret_cast<uint32_t*>(b + kv4_key_at(t, g, quarter, m)) = codes[0];
  if (it.four) {
    *reinterpret_cast<uint32_t*>(b + kv4_value_at(t & ~3, g, quarter * 4 + it.tok, m)) = run;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[kv4_value_at(t, g, quarter * 4 + i, m)] = (uint8_t)(codes[1] >> (8 * i));
  }
  if (quarter == 0) b[kv4_key_scale_at(t, g, m)] = (uint8_t)scale[0];
  if (quarter == 1) b[kv4_value_scale_at(t, g, m)] = (uint8_t)scale[1];
}

// ---- reading: the same way round ----------------------------------------------------------------------------------------
template <Elem E, int M>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Cache c, const int64_t* slots, int64_t rows, void* kout, void* vout, int vec) {
  typedef typename ElemOf<E>::T T;
  constexpr int m = M;   // (groups of 32: the offsets below become shifts and adds)
  Item it = item_of<M>(c, slots, rows);
  item_run(it);
  const int g = it.g, quarter = it.quarter, d0 = g * 32 + quarter * 8;
  uint32_t codes[2] = {0, 0}, scale[2] = {127, 127};
  if (it.live) {
    int t;
    const uint8_t* b = item_block(c, it, m, t);
    codes[0] = *reinterpret_cast<const uint32_t*>(b + kv4_key_at(t, g, quarter, m));
    scale[0] = b[kv4_key_scale_at(t, g, m)];
    scale[1] = b[kv4_value_scale_at(t, g, m)];
    if (it.four) {
      codes[1] = *reinterpret_cast<const uint32_t*>(b + kv4_value_at(t & ~3, g, quarter * 4 + it.tok, m));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) codes[1] |= (uint32_t)b[kv4_value_at(t, g, quarter * 4 + i, m)] << (8 * i);
    }
  }
  const uint32_t run = transpose4(codes[1], it.tok);
  if (it.four) codes[1] = run;
  if (it.r >= rows || it.h >= c.heads || d0 >= c.head_dim) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float s = kv4_scale(scale[w]);
    const uint32_t p[4] = {kv4_pair_bf16<0>(codes[w], s), kv4_pair_bf16<1>(codes[w], s), kv4_pair_bf16<2>(codes[w], s), kv4_pair_bf16<3>(codes[w], s)};
    T* o = static_cast<T*>(w ? vout : kout) + (it.r * c.heads + it.h) * c.head_dim + d0;
    if (vec) {   // four elements at a time: a head width is a multiple of four then
      if constexpr (E == Elem::bf16) {
        *reinterpret_cast<uint2*>(o) = uint2{p[0], p[1]};
        if (d0 + 8 <= c.head_dim) *reinterpret_cast<uint2*>(o + 4) = uint2{p[2], p[3]};
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(p[i] << 16), x[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
        store_elems<E, 4>(o, x);
        if (d0 + 8 <= c.head_dim) store_elems<E, 4>(o + 4, x + 4);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < c.head_dim) o[e] = ElemOf<E>::put(__uint_as_float(e & 1 ? p[e / 2] & 0xffff0000u : p[e / 2] << 16));
    }
  }
}

template <class F>
void by_groups(int m, F&& f) {
  switch (m) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    case 8: return f(std::integral_constant<int, 8>{});
    default: throw std::invalid_argument("4-bit cache: head width above 256");
  }
}
// whether four elements at a time may be read or written
bool by_fours(const void* p, std::initializer_list<int64_t> strides, int head_dim, size_t size) {
  if (head_dim % 4 != 0 || (uintptr_t)p % (4 * size) != 0) return false;
  for (int64_t s : strides)
    if (s % 4 != 0) return false;
  return true;
}

}  // namespace

void page_plan(int32_t* table, int batch, int width, const int32_t* kv_lens, const int32_t* new_lens, const int32_t* row_start,
               int64_t rows, const int32_t* free_pages, int64_t n_free, int page_shift, int64_t* slots, int32_t* used, hipStream_t s) {
  const Plan p{table, kv_lens, new_lens, row_start, free_pages, slots, used, rows, n_free, batch, width, page_shift};
  MSH_LAUNCH(page_plan_kernel, dim3(batch), dim3(256), 0, s, p);
}

void kv4_write(const Kv4Cache& c, const Kv4Rows& k, const Kv4Rows& v, Elem type, int64_t rows, const int64_t* slots, hipStream_t s) {
  if (rows == 0) return;
  const size_t size = elem_bytes(type);
  const int vec = k.elem == 1 && v.elem == 1 && by_fours(k.p, {k.row, k.head}, c.head_dim, size) && by_fours(v.p, {v.row, v.head}, c.head_dim, size);
  const dim3 grid((unsigned)kv4_rows_groups(rows), (unsigned)((c.heads * kv4_groups(c.head_dim) + 15) / 16));
  by_groups(kv4_groups(c.head_dim), [&](auto m) {
    constexpr int M = decltype(m)::value;
    if (type == Elem::f32) MSH_LAUNCH((kv4_write_kernel<Elem::f32, M>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
    else if (type == Elem::bf16) MSH_LAUNCH((kv4_write_kernel<Elem::bf16, M>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
    else MSH_LAUNCH((kv4_write_kernel<Elem::f16, M>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
  });
}

void kv4_read(const Kv4Cache& c, const int64_t* slots, int64_t rows, void* k, void* v, Elem type, hipStream_t s) {
  if (rows == 0) return;
  const size_t size = elem_bytes(type);
  const int vec = by_fours(k, {}, c.head_dim, size) && by_fours(v, {}, c.head_dim, size);
  const dim3 grid((unsigned)kv4_rows_groups(rows), (unsigned)((c.heads * kv4_groups(c.head_dim) + 15) / 16));
  by_groups(kv4_groups(c.head_dim), [&](auto m) {
    constexpr int M = decltype(m)::value;
    if (type == Elem::f32) MSH_LAUNCH((kv4_read_kernel<Elem::f32, M>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
    else if (type == Elem::bf16) MSH_LAUNCH((kv4_read_kernel<Elem::bf16, M>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
    else MSH_LAUNCH((kv4_read_kernel<Elem::f16, M>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
  });
}

// ---- attention: dispatch ------------------------------------------------------------------------------------------------
void kv4_attention_f32(const Kv4Attention& a, hipStream_t s);
void kv4_attention_bf16(const Kv4Attention& a, hipStream_t s);
void kv4_attention_f16(const Kv4Attention& a, hipStream_t s);

// Which form, by the rows of one key / value head and the work there is (times in us; 32 query over 8 key / value heads of 128, bf16, unless it says otherwise):
// * more than 64 rows: the form for chunks once its units of 128 rows fill the chip's 512 places (2048 tokens: 2 x 1024 queries 112 against 120 by
//   tiles of 32, 64 sequences of 512 with 128 queries each 133 against 202; half as many units: 1 x 1024 queries 80 against 70).  These are of 8 pairs of
//   sequence and head or a multiple; other numbers leave XCDs idle in this form (kv4_attention_chunk_kernel), which the rule does not weigh.
// * tiles of 32 once tiles of 16, four waves each, take more than half the places for waves (32 sequences of 2048, 20 rows: 27 against 29, 64 rows: 38 against
//   49; fp32, 4 heads of 64, 32 rows, 256 units of 16: 12.7 against 8.6) -- but not for fp32 rows of more than 64, which spill (64 rows: 70 by tiles of
//   16 against 76; 3 x 8 rows over 4 heads of 96, 128 sequences of 2000: 56 against 64).
// * tiles of 16: all four waves of a workgroup share a tile as long as there are too few to fill the chip's places for waves (1024 SIMDs) without,
//   then two, then none -- a wave's beginning and end cost as much as three blocks, so sooner for short tables and later for long ones (units, KW 4 / 2 / 1; fp32, two
//   places a SIMD, 10 tokens: 512 units 8.9 / 7.4 / 7.6, 1024 units 15 / 9.1 / 7.7; three places, 415 tokens: 1024 units 15.8 / 14.4 / 16.6, 2048
//   units 27 / 24 / 24; 2048 tokens: 1280 units 55 / 62 / 85, 1536 units 67 / 67 / 89, 4096 units 191 / 181 / 184).
Kv4Shape kv4_attention_shape(const Kv4Attention& a, Elem type) {
  const int groups = kv4_groups(a.cache.head_dim);
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads), pairs = (int64_t)a.batch * a.cache.heads;
  const int64_t units = pairs * ((rows + 15) / 16), room = (int64_t)a.width << a.cache.page_shift;
  const int64_t places = 1024 * kv4_attention_waves(groups, type == Elem::f32);
  if (a.fixed) return Kv4Shape{1, 4, false};
  if (rows > 64 && pairs * ((rows + 127) / 128) >= 512) return Kv4Shape{2, 4, true};
  if (rows > 16 && units * 8 > places && !(type == Elem::f32 && groups > 2)) return Kv4Shape{2, 4, false};
  const int64_t ample = room <= 128 ? places / 2 : room <= 1024 ? places : places * 2;
  return Kv4Shape{1, units * 4 <= ample ? 4 : units * 2 <= ample ? 2 : 1, false};
}

// Key ranges, joined by a second launch (4 to 40 us, by the rows).  The lengths live on the device; the host knows the table's room only.  A
// range is a share of each sequence's own length, so a short sequence in a wide table costs empty ranges and nothing else.
// Few units: as many ranges as fill the chip, none of them shorter than pays for its share of the join (single tokens, units x tokens, ranges 1 / 2 /
// 4 / 8 / 16 / 32: 8 x 1024: 11 / 10 / 9.1 / 8.5 / 9.0 / 10; 64 x 4096: 29 / 20 / 15 / 14 / 17 / 24; 128 x 16384: 107 / 61 / 51 / 49 / 52 / 62, but with
// lengths between 12001 and 40000 161 at 2, 116 at 8 and 106 at 16; 512 x 4096: 47 / 49 / 52 / 59; fp32 512 x 2048 32 / 40; 32-row tiles: 32 x 8192: 73 /
// 44 / 29 / 22 / 26 / 34; 256 x 2048: 27 / 32).  Below 1024 tokens one (8 units x 600: 8.4 / 9.7).
// Chunks: two ranges where units are few enough for long and short sequences to leave places empty at the end (4 sequences of 2500 to 8191 tokens,
// 485 to 1000 queries: 529 against 617; all of 8192: 771 against 752; at 2048 tokens the join would cost a quarter: 260 against 207).
// At most 32, so one sequence with few heads does not fill the chip (one token over 40000, 1 / 2 / 4 / 8 key / value heads: 15.7 / 15.7 / 15.6 / 16.6).
int kv4_attention_splits(const Kv4Attention& a, Elem type) {
  const Kv4Shape shape = kv4_attention_shape(a, type);
  if (a.fixed || shape.kw != 4 || kv4_join_groups(a.rows, a.heads) > kGroupsMost) return 1;
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads);
  const int64_t units = (int64_t)a.batch * a.cache.heads * ((rows + shape.rows() - 1) / shape.rows());
  const int64_t room = (int64_t)a.width << a.cache.page_shift;
  if (shape.chunk) return units < 1536 && room >= 8192 ? 2 : 1;
  if (room < 1024) return 1;
  const int64_t places = shape.rt == 2 ? 512 : 256 * kv4_attention_waves(kv4_groups(a.cache.head_dim), type == Elem::f32);   // for workgroups
  const int64_t wanted = room < 16384 ? places : places * 5 / 2;
  const int64_t least = units <= 32 ? 256 : (units <= 128 ? 512 : 2048) * shape.rt;
  int64_t n = wanted / units;
  n = n < room / least ? n : room / least;
  return (int)(n < 1 ? 1 : n > 32 ? 32 : n);
}
int64_t kv4_attention_groups(const Kv4Attention& a, Elem type) {
  const Kv4Shape shape = kv4_attention_shape(a, type);
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads), pairs = (int64_t)a.batch * a.cache.heads;
  const int64_t units = pairs * ((rows + shape.rows() - 1) / shape.rows()), per_group = 4 / shape.kw;
  return shape.chunk ? (pairs + 7) / 8 * 8 * (units / pairs) * a.nsplit : (units + per_group - 1) / per_group;   // (chunks: the second axis is in the first)
}
size_t kv4_attention_part_floats(const Kv4Attention& a, int nsplit) {
  return nsplit > 1 ? (size_t)a.rows * a.heads * nsplit * (32 * kv4_groups(a.cache.head_dim) + kPartPad) : 0;
}
void kv4_attention(const Kv4Attention& a, Elem type, hipStream_t s) {
  if (a.rows == 0 || a.batch == 0) return;
  if (type == Elem::f32) kv4_attention_f32(a, s);
  else if (type == Elem::bf16) kv4_attention_bf16(a, s);
  else kv4_attention_f16(a, s);
}

}  // namespace msh
