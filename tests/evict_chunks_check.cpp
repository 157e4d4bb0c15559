// Walks, on the host, how an eviction's chunks wait for each other (the function that the kernel calls), for lists drawn from a seed: whom a chunk waits for has
// been drawn before it, at most two of them, and they are all that read what it writes; by any order of steps every row gets where it belongs, and where chunks
// give up, what they leave is told.
//   evict_chunks_check seed
#include <algorithm>
#include <cstdio>
#include <cstdlib>
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

// `keep` of `length` places, ascending: at random, the first or last ones, or stretches.
static std::vector<int> list(int length, int keep) {
  std::vector<int> all(length), weight(length);
  const int kind = draw(0, 4), stretch = draw(1, 40);
  for (int i = 0; i < length; ++i) {
    all[i] = i;
    weight[i] = kind == 0 ? draw(0, 1 << 20) : kind == 1 ? -i : kind == 2 ? i : kind == 3 ? (i / stretch % 2) * 1000 + draw(0, 10) : (i < length / 3) * 1000 + draw(0, 500);
  }
  std::stable_sort(all.begin(), all.end(), [&](int a, int b) { return weight[a] > weight[b]; });
  all.resize(keep);
  std::sort(all.begin(), all.end());
  return all;
}

static int walk(bool give_up) {
  const int size = 1 << draw(0, 6), length = draw(2, 600), keep = draw(1, length - 1), chunks = (keep + size - 1) / size;
  const std::vector<int> kept = list(length, keep);
  std::vector<int> before(chunks + 1, -1000000);   // (the ones behind the length: nobody writes them)
  for (int i = 0; i <= chunks; ++i)
    if (i * size < length) before[i] = (int)(std::lower_bound(kept.begin(), kept.end(), i * size) - kept.begin());
  struct Chunk {
    int step = 0;   // 0: not drawn, 1: to read, 2: to look at others, 3: to write, 4: done
    bool gave_up = false, flag = false;
    EvictReaders readers{0, 0};
    std::vector<int> rows;
  };
  std::vector<Chunk> of(chunks);
  for (int c = 0; c < chunks; ++c) {
    const int first = c * size, count = std::min(size, keep - first);
    const EvictReaders r = of[c].readers = evict_readers(c, size, length, before.data());
    CHECK(r.first >= 0 && r.count >= 0 && r.count <= 2 && r.first + r.count <= c, "chunk %d of %d waits for %d + %d", c, chunks, r.first, r.count);
    for (int other = 0; other < chunks; ++other) {
      bool reads = false;
      for (int i = other * size; i < std::min(keep, (other + 1) * size); ++i) reads |= kept[i] >= first && kept[i] < first + size;
      if (other != c) CHECK(reads == (other >= r.first && other < r.first + r.count), "chunk %d of %d: %d reads there: %d", c, chunks, other, reads);
    }
    if (kept[first + count - 1] == first + count - 1) of[c].step = -1;   // (all of them are where they belong: nothing is read or said)
  }
  // any order of steps, chunks drawn in ascending order
  std::vector<int> row(length);
  for (int i = 0; i < length; ++i) row[i] = i;
  std::vector<int> told = kept;
  constexpr int kNaN = -7;
  int drawn = 0, done = 0;
  for (long long steps = 0; done < chunks; ++steps) {
    CHECK(steps < 10000000, "%d of %d chunks end", done, chunks);
    if (drawn < chunks && draw(0, 3) == 0) {
      Chunk& next = of[drawn++];
      if (next.step < 0) ++done, next.step = 4;
      else next.step = 1;
    }
    if (drawn == 0) continue;
    const int c = draw(0, drawn - 1), first = c * size, count = std::min(size, keep - first);
    Chunk& it = of[c];
    if (it.step == 1) {
      for (int i = 0; i < count; ++i) it.rows.push_back(row[kept[first + i]]);
      it.flag = true, it.step = 2;
    } else if (it.step == 2) {
      bool all = true;
      for (int i = 0; i < it.readers.count; ++i) all &= of[it.readers.first + i].flag;
      it.gave_up = !all && give_up && draw(0, 1);
      if (all || it.gave_up) it.step = 3;
    } else if (it.step == 3) {
      for (int i = 0; i < count; ++i) {
        row[first + i] = it.gave_up ? kNaN : it.rows[i];
        if (it.gave_up) told[first + i] = kEvictAbandoned;
      }
      it.step = 4, ++done;
    }
  }
  for (int i = 0; i < keep; ++i) {
    if (!give_up) CHECK(row[i] == kept[i] && told[i] == kept[i], "place %d of %d has %d, not %d", i, keep, row[i], kept[i]);
    else CHECK(told[i] == kEvictAbandoned ? row[i] == kNaN : told[i] == kept[i] && (row[i] == kept[i] || row[i] == kNaN), "place %d of %d has %d, the list %d", i, keep, row[i], told[i]);
  }
  return 0;
}

int main(int argc, char** argv) {
  if (argc != 2) return 2;
  rng.seed(std::atoi(argv[1]));
  for (int i = 0; i < 3000; ++i)
    if (walk(i % 3 == 0)) return 1;
  return 0;
}
