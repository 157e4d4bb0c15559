// The parts that rows of a paged cache are cut into (the functions that the kernels and their launch call), for lengths drawn from a seed.
//   paged_parts_check few    where all tiles can have a workgroup each, they do, whether sequences fill their tables or not
//   paged_parts_check many   no launch has fewer workgroups than parts; no part is longer than an even share and the least asks for
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "../intrasm_engine_amd/csrc/paged_cache.h"

using namespace iex;

static std::mt19937 rng;
static int draw(int low, int high) { return low + (int)(rng() % (unsigned)(high - low + 1)); }
#define CHECK(cond, ...)                                    \
  do {                                                      \
    if (!(cond)) { std::printf(__VA_ARGS__); std::printf("\n"); return 1; } \
  } while (0)

static int walk(int seqs, int width, int wanted, int few, bool full, bool all_few) {
  const int slots = (int)paged_slots(wanted, seqs, width);
  std::vector<int> tiles(seqs);
  int total = 0;
  for (int& t : tiles) total += t = full ? width : draw(1, width);
  if (slots == 0) return 0;   // (rows stay whole)
  const int least = paged_least(total, few), most = paged_part_most(total - seqs, slots, least);
  long long parts = 0;
  for (int t : tiles) {
    parts += paged_parts(t, most);
    if (all_few) CHECK(paged_parts(t, most) == t, "%d of %d tiles in %d parts (%d sequences, %d slots)", t, width, paged_parts(t, most), seqs, slots);
  }
  CHECK(parts <= (long long)seqs + slots, "%lld parts, %d sequences and %d slots", parts, seqs, slots);
  CHECK(most <= std::max(least, (total + slots - 1) / slots), "parts of %d tiles", most);
  return 0;
}

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  rng.seed(std::atoi(argv[2]));
  const bool few = !std::strcmp(argv[1], "few");
  for (int i = 0; i < 20000; ++i) {
    const int seqs = draw(1, few ? 40 : 3000), width = draw(1, few ? 64 : 2000), tiles = seqs * width;
    if (walk(seqs, width, few ? draw(tiles, 2 * tiles) : draw(0, 2000), few ? tiles : draw(0, 600), draw(0, 1), few)) return 1;
  }
  return 0;
}
