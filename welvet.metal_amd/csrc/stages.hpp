// stages.hpp — the order of a tile's copies into LDS (tiles.hpp): which step sends
// which, and how many may still be under way when a step reads its own.  Plain
// C++, so that a host program can replay it.  Internal to the library.
#pragma once

namespace wh {
namespace tiles {

// A product's sum runs in steps of one of A's `parts` each, `parts` of them over one
// stage of B.  A's steps take turns in `places_a` of LDS, B's stages in `places_b`, and
// at step h A is sent for places_a - 1 steps ahead, B, ahead of it, for places_b - 1
// stages.  Copies end in the order in which they were sent.
struct Stages {
  int parts, places_a, places_b;
  constexpr bool sends_a(int h, int steps) const { return h + places_a - 1 < steps; }
  constexpr bool sends_b(int h, int steps) const { return h % parts == 0 && h + (places_b - 1) * parts < steps; }
  // Copies of A and of B sent after those that a step of this part reads: of A the
  // steps' between, of B those that were sent with them.
  constexpr int left_a() const { return places_a - 2; }
  constexpr int left_b(int part) const {
    return places_b == 2 ? (parts == 2 && part == 1) : parts == 1 ? left_a() : (left_a() + part) / 2;
  }
  // Towards the end, where not all of these are sent any more, a step waits for every
  // copy.  Of six places each and two parts B, ten steps ahead, runs out before A.
  constexpr bool drains(int h, int steps) const {
    const int a = places_a + parts, b = (places_b - 1) * parts;
    return h + (a > b ? a : b) >= steps;
  }
};

}  // namespace tiles
}  // namespace wh
