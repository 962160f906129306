// The list in which a wave of the beam selection (k_beam.hip) keeps what can still be among the K best of its part: its room, and the
// two rules that keep it there.  Plain C++: tests/c/beam_list.cpp walks the same rules on the host.
#pragma once

namespace msh {

constexpr int kBeamMax = 16;
constexpr int kLane = 32;                                         // elements of a lane per chunk, 64 lanes
constexpr int kListMax = 2 * kBeamMax + kBeamMax * (kLane + 1);   // room for one chunk's most beside 2 K

// Before a chunk is added: whether the n entries there are have to be cut to the K best, so that K (kLane + 1) more have room.
constexpr bool beam_list_cut(int n, int K) { return n > kListMax - K * (kLane + 1); }

// Whether the bound has to rise to the K-th largest of the lanes' maxima before a chunk is added in which `over` lanes hold something
// above it.  It does until K elements are known to reach it (`enough`), and whenever those lanes could fill the list: each may bring kLane
// elements.  What a chunk adds is therefore in the room --
//   bound raised:      fewer than K lanes stay above it, (K - 1) kLane elements, and ties fill up to K:  at most K (kLane + 1)
//   over <= K lanes:   K kLane elements
//   otherwise:         n + over kLane <= kListMax, checked here
// Measured, us a call: raised for every chunk with more than K lanes above it, 256 x 8 beams over 32768 bf16 logits 56 instead of 53, 1 x 7 over 193263 19.5
// instead of 18.3; asked for less often, by a list of 900 entries, 1 x 16 over 193001 68 instead of 42 (longer lists to rank).
constexpr bool beam_bound_rises(int n, int K, int over, bool enough) { return over > K && (!enough || n + over * kLane > kListMax); }

}  // namespace msh
