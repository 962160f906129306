// The paged 4-bit cache: plan of pages and slots, writing rows, reading rows (form: serve_kernels.h).
#include "kv4_common.h"

namespace msh {
namespace {

// ---- plan ---------------------------------------------------------------------------------------------------------------
// need_b = ceil(len_b / P), kept_b = ceil((len_b - new_b) / P), first_b = sum of need - kept over the requests before b; table entry
// kept_b + i of request b becomes free[first_b + i], and the row at place p of request b the slot table[b][p / P] * P + p mod P.
// A few bytes per request: bound by the latency of its two launches.
struct Plan {
  int32_t* table;
  const int32_t *kv_lens, *new_lens, *row_start, *free_pages;
  int64_t* slots;
  int32_t *used, *first;
  int64_t rows, n_free;
  int32_t batch, width, page_shift;
};

__device__ __forceinline__ void plan_lens(const Plan& p, int b, int64_t& held, int64_t& fresh) {
  const int64_t most = (int64_t)p.width << p.page_shift;
  held = p.kv_lens[b], fresh = p.new_lens[b];
  held = held < 0 ? 0 : held > most ? most : held;
  fresh = fresh < 0 ? 0 : fresh > held ? held : fresh;
}
__device__ __forceinline__ int pages_of(int64_t tokens, int shift) { return (int)((tokens + (1 << shift) - 1) >> shift); }

// pages taken by the requests before `b`, summed by the whole workgroup (256 threads; every request's lengths are 8 bytes)
__device__ int64_t plan_before(const Plan& p, int b, int64_t* red) {
  int64_t sum = 0;
  for (int i = threadIdx.x; i < b; i += 256) {
    int64_t held, fresh;
    plan_lens(p, i, held, fresh);
    sum += pages_of(held, p.page_shift) - pages_of(held - fresh, p.page_shift);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// one workgroup per request: its table row, then the slots of its rows
__global__ __launch_bounds__(256) void page_plan_kernel(Plan p) {
  __shared__ int64_t red[4];
  const int b = blockIdx.x;
  const int64_t first = plan_before(p, b, red);
  int64_t held, fresh;
  plan_lens(p, b, held, fresh);
  const int kept = pages_of(held - fresh, p.page_shift), need = pages_of(held, p.page_shift);
  if (b == p.batch - 1 && threadIdx.x == 0) *p.used = (int32_t)(first + need - kept);
  int32_t* row = p.table + (int64_t)b * p.width;
  auto page_at = [&](int c) -> int32_t {
    if (c < kept) return row[c];
    const int64_t at = first + c - kept;
    return c < need && at < p.n_free ? p.free_pages[at] : -1;
  };
  const int64_t start = p.row_start[b];
  for (int64_t i = threadIdx.x; i < fresh; i += 256) {   // reads of kept entries only, which no thread of the grid writes
    const int64_t at = start + i, place = held - fresh + i;
    if (at < 0 || at >= p.rows) continue;
    const int32_t page = page_at((int)(place >> p.page_shift));
    p.slots[at] = page < 0 ? -1 : ((int64_t)page << p.page_shift) + (place & ((1 << p.page_shift) - 1));
  }
  for (int c = kept + threadIdx.x; c < p.width; c += 256) row[c] = page_at(c);
}

__global__ __launch_bounds__(256) void page_plan_clear_kernel(int64_t* slots, int64_t rows) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < rows) slots[i] = -1;
}

// ---- writing ------------------------------------------------------------------------------------------------------------
// e = floor(log2(amax)) - 2, one more where the mantissa is 1.75 or above: amax / 2^e lies in [3.5, 7), and what saturates at 6 or
// rounds at 3.5 is off by a seventh at most.  NaN is stored as 0, infinities as the largest finite value.
__device__ __forceinline__ float storable(float x) {
  x = x != x ? 0.f : x;
  return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
}
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x200000u) >> 23) - 129;
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

// four neighbouring threads hold a group of 32 elements
template <Elem E>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4Cache c, Kv4Rows k, Kv4Rows v, int64_t rows, const int64_t* slots, int vec) {
  typedef typename ElemOf<E>::T T;
  const int m = kv4_groups(c.head_dim);
  const int per = c.heads * m * 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = id / per;
  const int in = (int)(id % per), quarter = in & 3, g = (in >> 2) % m, h = (in >> 2) / m;
  int64_t slot = r < rows ? slots[r] : -1;
  if (slot >= c.pages << c.page_shift) slot = -1;
  const int d0 = g * 32 + quarter * 8;
  float x[2][8];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const Kv4Rows& src = w ? v : k;
    const T* p = static_cast<const T*>(src.p) + r * src.row + h * src.head + d0 * src.elem;
    if (slot >= 0 && vec && d0 + 8 <= c.head_dim) {
      load_elems<E, 8>(p, x[w]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[w][e] = slot >= 0 && d0 + e < c.head_dim ? ElemOf<E>::get(p[e * src.elem]) : 0.f;
    }
  }
  uint32_t codes[2], scale[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[w][e] = storable(x[w][e]), a = fmaxf(a, fabsf(x[w][e]));
    a = fmaxf(a, __shfl_xor(a, 1));
    a = fmaxf(a, __shfl_xor(a, 2));
    scale[w] = scale_byte(a);
    codes[w] = codes8(x[w], kv4_scale(scale[w]));
  }
  if (slot < 0) return;
  const int64_t page = slot >> c.page_shift;
  const int place = (int)(slot & ((1 << c.page_shift) - 1)), t = place & 31;
  uint8_t* b = c.data + (((page * c.heads + h) << (c.page_shift - 5)) + (place >> 5)) * kv4_block_bytes(m);
  *reinterpret_cast<uint32_t*>(b + kv4_key_at(t, g, quarter, m)) = codes[0];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[kv4_value_at(t, g, quarter * 4 + i, m)] = (uint8_t)(codes[1] >> (8 * i));
  if (quarter == 0) b[kv4_key_scale_at(t, g, m)] = (uint8_t)scale[0];
  if (quarter == 1) b[kv4_value_scale_at(t, g, m)] = (uint8_t)scale[1];
}

// ---- reading ------------------------------------------------------------------------------------------------------------
template <Elem E>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Cache c, const int64_t* slots, int64_t rows, void* kout, void* vout, int vec) {
  typedef typename ElemOf<E>::T T;
  const int m = kv4_groups(c.head_dim);
  const int per = c.heads * m * 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = id / per;
  if (r >= rows) return;
  const int in = (int)(id % per), quarter = in & 3, g = (in >> 2) % m, h = (in >> 2) / m;
  const int64_t slot = slots[r];
  const int d0 = g * 32 + quarter * 8;
  if (d0 >= c.head_dim) return;
  uint32_t codes[2] = {0, 0}, scale[2] = {127, 127};
  if (slot >= 0 && slot < c.pages << c.page_shift) {
    const int64_t page = slot >> c.page_shift;
    const int place = (int)(slot & ((1 << c.page_shift) - 1)), t = place & 31;
    const uint8_t* b = c.data + (((page * c.heads + h) << (c.page_shift - 5)) + (place >> 5)) * kv4_block_bytes(m);
    codes[0] = *reinterpret_cast<const uint32_t*>(b + kv4_key_at(t, g, quarter, m));
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[1] |= (uint32_t)b[kv4_value_at(t, g, quarter * 4 + i, m)] << (8 * i);
    scale[0] = b[kv4_key_scale_at(t, g, m)];
    scale[1] = b[kv4_value_scale_at(t, g, m)];
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float s = kv4_scale(scale[w]);
    uint32_t p[4] = {kv4_pair_bf16<0>(codes[w], s), kv4_pair_bf16<1>(codes[w], s), kv4_pair_bf16<2>(codes[w], s), kv4_pair_bf16<3>(codes[w], s)};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(p[i] << 16), x[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
    T* o = static_cast<T*>(w ? vout : kout) + (r * c.heads + h) * c.head_dim + d0;
    if (vec && d0 + 8 <= c.head_dim) {
      store_elems<E, 8>(o, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (d0 + e < c.head_dim) o[e] = ElemOf<E>::put(x[e]);
    }
  }
}

unsigned grid_of(int64_t threads) { return (unsigned)((threads + 255) / 256); }
bool aligned16(const void* p, std::initializer_list<int64_t> strides, size_t size) {
  if ((uintptr_t)p % 16 != 0) return false;
  for (int64_t s : strides)
    if (s * (int64_t)size % 16 != 0) return false;
  return true;
}

}  // namespace

void page_plan(int32_t* table, int batch, int width, const int32_t* kv_lens, const int32_t* new_lens, const int32_t* row_start,
               int64_t rows, const int32_t* free_pages, int64_t n_free, int page_shift, int64_t* slots, int32_t* used, hipStream_t s) {
  Plan p{table, kv_lens, new_lens, row_start, free_pages, slots, used, nullptr, rows, n_free, batch, width, page_shift};
  if (rows > 0) MSH_LAUNCH(page_plan_clear_kernel, dim3(grid_of(rows)), dim3(256), 0, s, slots, rows);
  MSH_LAUNCH(page_plan_kernel, dim3(batch), dim3(256), 0, s, p);
}

void kv4_write(const Kv4Cache& c, const Kv4Rows& k, const Kv4Rows& v, Elem type, int64_t rows, const int64_t* slots, hipStream_t s) {
  if (rows == 0) return;
  const size_t size = elem_bytes(type);
  const int vec = k.elem == 1 && v.elem == 1 && aligned16(k.p, {k.row, k.head}, size) && aligned16(v.p, {v.row, v.head}, size);
  const dim3 grid(grid_of(rows * c.heads * kv4_groups(c.head_dim) * 4));
  if (type == Elem::f32) MSH_LAUNCH((kv4_write_kernel<Elem::f32>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
  else if (type == Elem::bf16) MSH_LAUNCH((kv4_write_kernel<Elem::bf16>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
  else MSH_LAUNCH((kv4_write_kernel<Elem::f16>), grid, dim3(256), 0, s, c, k, v, rows, slots, vec);
}

void kv4_read(const Kv4Cache& c, const int64_t* slots, int64_t rows, void* k, void* v, Elem type, hipStream_t s) {
  if (rows == 0) return;
  const size_t size = elem_bytes(type);
  const int vec = aligned16(k, {c.head_dim}, size) && aligned16(v, {c.head_dim}, size);
  const dim3 grid(grid_of(rows * c.heads * kv4_groups(c.head_dim) * 4));
  if (type == Elem::f32) MSH_LAUNCH((kv4_read_kernel<Elem::f32>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
  else if (type == Elem::bf16) MSH_LAUNCH((kv4_read_kernel<Elem::bf16>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
  else MSH_LAUNCH((kv4_read_kernel<Elem::f16>), grid, dim3(256), 0, s, c, slots, rows, k, v, vec);
}

// ---- attention: dispatch ------------------------------------------------------------------------------------------------
void kv4_attention_f32(const Kv4Attention& a, hipStream_t s);
void kv4_attention_bf16(const Kv4Attention& a, hipStream_t s);
void kv4_attention_f16(const Kv4Attention& a, hipStream_t s);

// The lengths live on the device; the host knows the table's room only.  A range is a share of each sequence's own length, so a short
// sequence in a wide table costs empty ranges and nothing else.
int kv4_attention_splits(const Kv4Attention& a, Elem type) {
  const int64_t rows = (int64_t)a.max_q * (a.heads / a.cache.heads);
  if (rows > 64) return 1;
  const int64_t groups = (int64_t)a.batch * a.cache.heads * ((rows + 31) / 32);
  const int64_t room = (int64_t)a.width << a.cache.page_shift;
  const int64_t most = (room + 255) / 256;   // two blocks per wave at least
  int64_t n = (2048 + groups - 1) / groups;
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
size_t kv4_attention_part_floats(const Kv4Attention& a, int nsplit) {
  return nsplit > 1 ? (size_t)a.rows * a.heads * nsplit * (32 * kv4_groups(a.cache.head_dim) + 2) : 0;
}
void kv4_attention(const Kv4Attention& a, Elem type, hipStream_t s) {
  if (a.rows == 0 || a.batch == 0) return;
  if (type == Elem::f32) kv4_attention_f32(a, s);
  else if (type == Elem::bf16) kv4_attention_bf16(a, s);
  else kv4_attention_f16(a, s);
}

}  // namespace msh
