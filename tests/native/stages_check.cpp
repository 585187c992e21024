// Replays the copies of a tile (csrc/stages.hpp, csrc/tiles.hpp) for sums of every
// length: at each step, what it reads has to have ended by its own wait, and what it
// sends must not take a place that is still to be read.
//   stages_check PARTS PLACES_A PLACES_B LOADS_A LOADS_B MOST_STAGES
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "stages.hpp"

using wh::tiles::Stages;

namespace {

struct Copy {
  bool b;  // of B
  int at;  // the step of A, the stage of B
};

// How many of `sent`, oldest first, have ended when at most `left` loads are under way;
// a copy's loads count one by one.
size_t ended(const std::vector<Copy> &sent, int loads_a, int loads_b, int left) {
  size_t n = sent.size();
  while (n > 0 && left >= (sent[n - 1].b ? loads_b : loads_a)) left -= sent[--n].b ? loads_b : loads_a;
  return left > 0 && n > 0 ? n - 1 : n;  // of the next one some are under way
}

bool replay(const Stages &s, int loads_a, int loads_b, int stages) {
  const int steps = stages * s.parts;
  std::vector<Copy> sent;
  for (int h = 0; h < s.places_a - 1; ++h) {
    if (h % s.parts == 0 && h / s.parts < s.places_b - 1 && h / s.parts < stages) sent.push_back({true, h / s.parts});
    if (h < steps) sent.push_back({false, h});
  }
  for (int b = (s.places_a - 2) / s.parts + 1; b < s.places_b - 1; ++b)
    if (b < stages) sent.push_back({true, b});
  std::vector<int> read_a(s.places_a, -1), read_b(s.places_b, -1);  // the last of each place that was read
  for (int h = 0; h < steps; ++h) {
    const int stage = h / s.parts;
    const size_t done = s.drains(h, steps) ? sent.size()
                                           : ended(sent, loads_a, loads_b, s.left_a() * loads_a + s.left_b(h % s.parts) * loads_b);
    bool a = false, b = false;
    for (size_t i = 0; i < done; ++i) {
      a |= !sent[i].b && sent[i].at == h;
      b |= sent[i].b && sent[i].at == stage;
    }
    if (!a || !b) {
      std::printf("parts %d places %d %d loads %d %d: step %d of %d reads %s that may be under way\n", s.parts,
                  s.places_a, s.places_b, loads_a, loads_b, h, steps, a ? "a stage of B" : "a step of A");
      return false;
    }
    // sent past the barrier: everything before this step has been read
    const auto send = [&](bool of_b, int at, int places, const std::vector<int> &read) {
      if (at - places >= 0 && read[at % places] != at - places) return false;
      sent.push_back({of_b, at});
      return true;
    };
    bool free = true;
    if (s.sends_b(h, steps)) free &= send(true, stage + s.places_b - 1, s.places_b, read_b);
    if (s.sends_a(h, steps)) free &= send(false, h + s.places_a - 1, s.places_a, read_a);
    read_a[h % s.places_a] = h;
    if (h % s.parts == s.parts - 1) read_b[stage % s.places_b] = stage;
    if (!free) {
      std::printf("parts %d places %d %d: step %d of %d sends into a place that is still read\n", s.parts, s.places_a,
                  s.places_b, h, steps);
      return false;
    }
  }
  if ((int)sent.size() != steps + stages) {
    std::printf("parts %d places %d %d: %zu copies of %d\n", s.parts, s.places_a, s.places_b, sent.size(), steps + stages);
    return false;
  }
  return true;
}

}  // namespace

int main(int argc, char **argv) {
  if (argc != 7) return 2;
  int v[6];
  for (int i = 0; i < 6; ++i) v[i] = std::atoi(argv[i + 1]);
  const Stages s{v[0], v[1], v[2]};
  for (int stages = 1; stages <= v[5]; ++stages)
    if (!replay(s, v[3], v[4], stages)) return 1;
  std::printf("stages_check: ok\n");
  return 0;
}
