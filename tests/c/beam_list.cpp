// A wave's pass over one part of a row, as beam_partial_kernel (csrc/k_beam.hip) makes it, on the host: the same chunks, lanes, order and
// -- through csrc/beam_list.h -- the same rules for the bound and the list's room.  Every write behind that room is counted.
#include <math.h>

#include <algorithm>
#include <vector>

#include "beam_list.h"

using namespace msh;

struct Entry {
  float val;
  int idx;
};
static bool before(const Entry& a, const Entry& b) { return a.val > b.val || (a.val == b.val && a.idx < b.idx); }

// x: the row; it starts `off` elements into its first vector of `vec` elements.  Part `part` of `parts` -> its K best in order (val, idx),
// how many there are, and the list's greatest length.
extern "C" int beam_list_walk(const float* x, int vocab, int vec, int off, int parts, int part, int K, float* val, int* idx, int* longest) {
  const int loads = kLane / vec, nv = (vocab + off + vec - 1) / vec, per = ((nv + parts - 1) / parts + 63) & ~63;
  const int v0 = part * per, v1 = std::min(v0 + per, nv);
  std::vector<Entry> list;
  float bound = -INFINITY;
  bool enough = false;
  *longest = 0;
  auto cut = [&] {
    std::sort(list.begin(), list.end(), before);
    if ((int)list.size() > K) list.resize(K);
  };
  for (int base = v0; base < v1; base += 64 * loads) {
    float e[64][kLane], hi[64];
    int at[64][kLane];
    for (int lane = 0; lane < 64; ++lane) {
      hi[lane] = -INFINITY;
      for (int i = 0; i < kLane; ++i) {
        const int v = base + (i / vec) * 64 + lane;
        at[lane][i] = v * vec + i % vec - off;
        e[lane][i] = v < v1 && at[lane][i] >= 0 && at[lane][i] < vocab ? x[at[lane][i]] : -INFINITY;
        hi[lane] = std::max(hi[lane], e[lane][i]);
      }
    }
    auto lanes_over = [&] { return (int)std::count_if(hi, hi + 64, [&](float h) { return h > bound; }); };
    int over = lanes_over();
    if (over == 0) continue;
    if (beam_list_cut((int)list.size(), K)) {
      cut();
      if ((int)list.size() == K) bound = std::max(bound, list[K - 1].val), enough = true;
      over = lanes_over();
    }
    const bool raise = beam_bound_rises((int)list.size(), K, over, enough);
    if (raise) {
      std::vector<float> h(hi, hi + 64);
      std::sort(h.begin(), h.end(), [](float a, float b) { return a > b; });
      if (!(h[K - 1] > bound)) return -1;   // the bound only ever rises
      bound = h[K - 1];
    }
    const size_t n0 = list.size();
    for (int lane = 0; lane < 64; ++lane)
      for (int i = 0; i < kLane; ++i)
        if (e[lane][i] > bound) list.push_back(Entry{e[lane][i], at[lane][i]});
    if (raise) {
      int after = -1;
      for (int k = (int)(list.size() - n0); k < K; ++k) {
        int next = 1 << 30;
        for (int lane = 0; lane < 64; ++lane)
          for (int i = 0; i < kLane; ++i)
            if (e[lane][i] == bound && at[lane][i] > after) next = std::min(next, at[lane][i]);
        if (next == 1 << 30) break;
        list.push_back(Entry{bound, next});
        after = next;
      }
      enough = true;
    }
    *longest = std::max(*longest, (int)list.size());
  }
  cut();
  for (size_t i = 0; i < list.size(); ++i) val[i] = list[i].val, idx[i] = list[i].idx;
  return (int)list.size();
}

extern "C" int beam_list_room() { return kListMax; }
