// Walks, on the host, what the kernels of the paged cache touch (the same functions that the device code calls), for sequences,
// offsets, tables and lists drawn from a seed, unsound ones among them, and reports the first access outside an array, token that
// is met twice or not at all, or workgroup that the launch has no room for.
//   paged_cache_check append|attend|keys seed
#include <algorithm>
#include <cmath>
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

static int append() {
  const int shift = draw(4, 8), page = 1 << shift, span = append_span(page), seqs = draw(0, 70), width = draw(0, 9), most = width << shift;
  const bool unsound = draw(0, 3) == 0, single = draw(0, 3) == 0;
  std::vector<int> offsets(seqs + 1, 0), lengths(seqs);
  int tokens = 0;
  for (int s = 0; s < seqs; ++s) {
    const int count = single ? 1 : draw(0, 3) == 0 ? 0 : draw(0, most > 0 ? most : 3);
    offsets[s + 1] = tokens += count;
    lengths[s] = count + (most > count ? draw(0, most - count) : 0);
    if (draw(0, 9) == 0) lengths[s] = draw(-5, most + 200);
  }
  if (!single) tokens += draw(0, 1) * draw(0, 200);
  if (unsound && !single)
    for (int& o : offsets)
      if (draw(0, 4) == 0) o = draw(-100, tokens + 100);
  if (unsound)
    for (int& l : lengths)
      if (draw(0, 4) == 0) l = (int)rng();
  const long long grid = single ? tokens : append_most_spans(tokens, seqs, span);
  std::vector<int> met(tokens + 1, 0);
  long long items = 0;
  for (int s = 0; s <= seqs; ++s) {
    if (single && s == seqs) break;
    const Appended a = single ? appended(s, seqs, tokens, s, s + 1, lengths[s], most)
                              : appended(s, seqs, tokens, offsets[s], s < seqs ? offsets[s + 1] : 0, s < seqs ? lengths[s] : 0, most);
    CHECK(a.first >= 0 && a.count >= 0 && a.first + a.count <= tokens, "sequence %d: tokens %d + %d of %d", s, a.first, a.count, tokens);
    CHECK(!a.sound || (a.position >= 0 && a.position + a.count <= most), "sequence %d: positions %d + %d of %d", s, a.position, a.count, most);
    const int spans = append_spans(a, span);
    CHECK(!single || spans == 1, "one token in %d spans", spans);
    for (int i = 0; i < spans; ++i, ++items) {
      if (items >= grid) { CHECK(unsound, "span %lld of %lld workgroups", items, grid); continue; }
      const int begin = (a.position / span + i) * span, low = a.position > begin ? a.position - begin : 0;
      const int end = a.position + a.count - begin, high = end < span ? end : span;
      CHECK(low < high, "sequence %d span %d is empty", s, i);
      for (int row = low; row < high; ++row) {
        const int position = begin + row, token = a.first + position - a.position;
        CHECK(token >= a.first && token < a.first + a.count, "token %d outside %d + %d", token, a.first, a.count);
        ++met[token];
        if (a.sound) CHECK(position >> shift < width, "entry %d of %d", position >> shift, width);
      }
    }
  }
  if (!unsound)
    for (int t = 0; t < tokens; ++t) CHECK(met[t] == 1, "token %d met %d times", t, met[t]);
  return 0;
}

static int attend() {
  const int shift = draw(4, 8), page = 1 << shift, seqs = draw(1, 150), width = draw(0, 4) == 0 ? draw(0, 2) : draw(1, 60), pages = draw(1, 50);
  const int count = draw(0, 1) ? 0 : draw(1, 20), few = draw(0, 400), entries = count ? count : width;
  std::vector<int> lengths(seqs), tokens(seqs);
  for (int& l : lengths) l = draw(0, 9) == 0 ? (int)rng() : draw(0, width * page);
  const int slots = draw(0, 5) == 0 ? 0 : (int)paged_slots(draw(0, 300), seqs, paged_tiles(entries * page));
  // parts of every row: whole rows, listed pages; 0: by the lengths
  const int longest = paged_tiles(entries * page), fixed = slots == 0 ? 1 : count ? paged_parts(longest, paged_part_most(seqs * longest, slots, paged_least(seqs * longest, few))) : 0;
  const int grid = fixed ? seqs * fixed : seqs + slots;
  CHECK(!fixed || fixed <= 1 + slots / seqs, "%d parts, %d slots for %d", fixed, slots, seqs);
  int total = 0;
  for (int s = 0; s < seqs; ++s) {
    const int n = cached_length(lengths[s], width, page);
    CHECK(n >= 0 && n <= width * page, "length %d of %d", n, width * page);
    tokens[s] = count && n ? count * page : n;
    total += paged_tiles(tokens[s]);
  }
  const int most = paged_part_most(fixed ? seqs * longest : total, slots, paged_least(fixed ? seqs * longest : total, few));
  int items = 0;
  for (int s = 0; s < seqs; ++s) {
    const int tiles = paged_tiles(fixed && count ? count * page : tokens[s]), parts = fixed ? fixed : paged_parts(tiles, most), n = cached_length(lengths[s], width, page);
    std::vector<int> table(width), list(count), met(tokens[s] + 1, 0);
    for (int& p : table) p = draw(0, 5) == 0 ? (int)rng() : draw(0, pages - 1);
    for (int& p : list) p = draw(0, 5) == 0 ? (int)rng() : draw(0, width);
    CHECK(paged_part_begin(tiles, parts, 0) == 0 && paged_part_begin(tiles, parts, parts) == tiles, "%d parts of %d tiles", parts, tiles);
    for (int i = 0; i < parts; ++i, ++items) {
      const int from = paged_part_begin(tiles, parts, i), to = paged_part_begin(tiles, parts, i + 1);
      CHECK(from < to && to - from <= most, "part of %d tiles, at most %d", to - from, most);
      const int begin = from * kPagedTile, end = std::min(tokens[s], to * kPagedTile), waves = draw(0, 2) ? 4 << draw(0, 1) : 1, places = draw(0, 1) ? 2 : 4;
      for (int wave = 0; wave < waves; ++wave)
        for (int t = begin + wave * places * 16; t < end; t += waves * places * 16)
          for (int a = 0; a < places; ++a) {
            const PagedPlace place = paged_place(t + a * 16, shift);
            CHECK(place.slot % 16 == 0 && place.slot + 16 <= page, "slot %d of %d", place.slot, page);
            if (place.entry >= entries) continue;
            const int logical = count ? list[place.entry] : place.entry;
            const int at = (unsigned)logical < (unsigned)width ? table[logical] : -1;
            const int valid = paged_valid((unsigned)logical < (unsigned)width ? logical : 0, place.slot, shift, at, pages, n);
            CHECK(valid >= 0 && valid <= 16 && (valid == 0 || (at >= 0 && at < pages)), "page %d of %d", at, pages);
            for (int x = 0; x < 16 && t + a * 16 + x < tokens[s]; ++x) ++met[t + a * 16 + x];
            if (!count && at >= 0 && at < pages) CHECK(valid == std::max(0, std::min(16, n - (t + a * 16))), "%d attended to", valid);
          }
    }
    for (int t = 0; t < tokens[s]; ++t) CHECK(met[t] == 1, "sequence %d token %d met %d times", s, t, met[t]);
  }
  CHECK(items <= grid, "%d parts in %d workgroups", items, grid);
  return 0;
}

static int keys() {
  auto bits = [](float x) { unsigned u; std::memcpy(&u, &x, 4); return u; };
  const float a = std::ldexp((float)draw(-1000, 1000) / 7.f, draw(-40, 40)), b = std::ldexp((float)draw(-1000, 1000) / 7.f, draw(-40, 40));
  CHECK((a < b) == (select_key(bits(a)) < select_key(bits(b))) && (a == b) == (select_key(bits(a)) == select_key(bits(b))), "%g and %g", a, b);
  CHECK(select_key(bits(-INFINITY)) > 0 && select_key(bits(-INFINITY)) < select_key(bits(-3e38f)) && select_key(bits(0.f)) == select_key(bits(-0.f)), "ends");
  CHECK(select_key(bits(INFINITY)) < kSelectNaN && select_key(bits(NAN)) == kSelectNaN && select_key(bits(-NAN)) == kSelectNaN && kSelectNaN < kSelectAlways, "order");
  const int e = e4m3_exponent(bits(std::fabs(a)));
  CHECK(a == 0 || (std::fabs(a) <= std::ldexp(448.0, e - 127) && std::fabs(a) > std::ldexp(224.0, e - 127)), "exponent %d of %g", e, a);
  const float edge = std::ldexp(448.f, draw(-30, 30));
  CHECK(edge == std::ldexp(448.0, e4m3_exponent(bits(edge)) - 127) && e4m3_exponent(bits(std::nextafter(edge, 1e38f))) == e4m3_exponent(bits(edge)) + 1, "edge %g", edge);
  CHECK(e4m3_exponent(0) == 1 && e4m3_exponent(bits(INFINITY)) <= 254 && e4m3_exponent(bits(1e-45f)) == 1, "extremes");
  return 0;
}

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  rng.seed(std::atoi(argv[2]));
  for (int i = 0; i < 3000; ++i) {
    const int rc = !std::strcmp(argv[1], "append") ? append() : !std::strcmp(argv[1], "attend") ? attend() : keys();
    if (rc) { std::printf("draw %d\n", i); return rc; }
  }
  return 0;
}
