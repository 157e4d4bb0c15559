// Which tokens, pages and rows the kernels of the paged cache (kv_append, paged_attention, select_pages) touch: how new
// tokens are dealt to workgroups, how a cache's length is split, where a page lies.  Plain C++, so that a program on the host
// can walk what it gives (tests/paged_cache_check.cpp, tests/paged_parts_check.cpp); the addresses that kernels make of it are theirs.  Lengths,
// offsets, tables and lists are device data that nobody has checked: everything here keeps inside the arrays whatever they hold.
#pragma once
#include <cstddef>

#include "gemm_addresses.h"   // IEX_HD

namespace iex {

// ---- lengths --------------------------------------------------------------------------------------------------------
// Tokens of a sequence that its table can hold.
IEX_HD int cached_length(int length, int table_width, int page_size) {
  const int most = table_width * page_size;   // (checked to fit on the host)
  return length < 0 ? 0 : length > most ? most : length;
}

// ---- attention: rows in parts -----------------------------------------------------------------------------------------
// A row is a sequence with one block of up to 16 query heads of a key head.  Rows of more than a certain number of tiles are cut
// into equal parts, a workgroup each; an empty sequence is one part too, which writes its zeros.
constexpr int kPagedTile = 128;   // tokens

IEX_HD int paged_tiles(int tokens) { return tokens <= kPagedTile ? 1 : tokens / kPagedTile + (tokens % kPagedTile != 0); }

// Tiles that a part has at most, where `beyond` tiles (of all sequences, one block of heads, beyond the first of each) go to `slots`
// workgroups.  The parts of all sequences are at most `slots` more than there are sequences: t tiles are 1 + (t - 1) / most parts at most.
IEX_HD int paged_part_most(int beyond, int slots, int least) {
  if (slots == 0) return 1 << 30;
  const int even = beyond / slots + (beyond % slots != 0);
  return even > least ? even : least;
}
// The `least` above, of all tiles: one where each (at most `few`) can have a workgroup, else two.
IEX_HD int paged_least(int total, int few) { return total <= few ? 1 : 2; }
IEX_HD int paged_parts(int tiles, int most) { return tiles <= most ? 1 : tiles / most + (tiles % most != 0); }
// The first tile of a part (of part number `parts`: the end).
IEX_HD int paged_part_begin(int tiles, int parts, int part) { return (int)((long long)tiles * part / parts); }

// Slots that are worth having: none where no sequence can be long enough to be cut.
IEX_HD long long paged_slots(long long wanted, long long seqs, int most_tiles) {
  const long long most = seqs * (most_tiles - 1);
  return most < wanted ? (most < 0 ? 0 : most) : wanted < 1 ? 1 : wanted;
}

// Where 16 tokens of a sequence from `token` on lie (16 divides token and the page): entry `entry` of the sequence's table (or
// list of pages), first slot in the page.
struct PagedPlace {
  int entry, slot;
};
IEX_HD PagedPlace paged_place(int token, int page_shift) { return PagedPlace{token >> page_shift, token & ((1 << page_shift) - 1)}; }

// How many of the 16 tokens from `slot` of the sequence's page `logical` on it attends to.  `page`: where that page lies, as the
// table says; outside the cache: given back, nothing of it is attended to (or read).
IEX_HD int paged_valid(int logical, int slot, int page_shift, int page, int pages, int length) {
  if ((unsigned)page >= (unsigned)pages) return 0;
  const int left = length - ((logical << page_shift) + slot);
  return left < 0 ? 0 : left > 16 ? 16 : left;
}

// ---- appending: new tokens in spans -----------------------------------------------------------------------------------
// A span is an aligned stretch of positions of one sequence, whole pages of it.
IEX_HD int append_span(int page_size) { return page_size > 64 ? page_size : 64; }

// The new tokens of one sequence: tokens first .. first + count of the call at positions from `position` on.  Not `sound`: it
// has no place for them (a length beyond its table or short of its new tokens); they are passed over.
struct Appended {
  int first, count, position, sound;
};
// offsets == nullptr: one token per sequence.  Sequence number `seqs` stands for the tokens behind the last sequence's.
IEX_HD Appended appended(int s, int seqs, int tokens, int begin, int end, int length, int most) {
  if (s > seqs) return Appended{0, 0, 0, false};
  if (s == seqs) end = tokens;
  if (begin < 0) begin = 0;
  if (begin > tokens) begin = tokens;
  if (end > tokens) end = tokens;
  const int count = end > begin ? end - begin : 0;
  const bool sound = s < seqs && length <= most && length >= count;
  return Appended{begin, count, sound ? length - count : 0, sound};
}
IEX_HD int append_spans(const Appended& a, int span) {
  return a.count == 0 ? 0 : (a.position + a.count - 1) / span - a.position / span + 1;
}
// Spans that a launch has workgroups for: every sequence with new tokens has one more than its whole spans, at most two more
// (and the tokens behind the last sequence are like one sequence more); none is empty.
IEX_HD long long append_most_spans(long long tokens, long long seqs, int span) {
  const long long with = seqs + 1 < tokens ? seqs + 1 : tokens;
  const long long spans = tokens / span + 2 * with;
  return spans < tokens ? spans : tokens;
}

// ---- e4m3 -------------------------------------------------------------------------------------------------------------
// The exponent of a row whose largest magnitude has these bits (as fp32): the least power of two, biased by 127, that brings it
// to 448, e4m3's largest value.  (Of a row's finite values: its infinities and NaN become NaN.)
IEX_HD int e4m3_exponent(unsigned magnitude_bits) {
  const int e = (int)((magnitude_bits + 0x1FFFFFu) >> 23) - 8;   // (mantissas above 1.75 round up)
  return e < 1 ? 1 : e > 254 ? 254 : e;
}

// ---- selection --------------------------------------------------------------------------------------------------------
// Scores as whole numbers in the same order: 0 for a page that cannot be selected, the largest for one that has to be, the next
// for NaN.
constexpr unsigned kSelectAlways = 0xFFFFFFFFu, kSelectNaN = 0xFFFFFFFEu;
IEX_HD unsigned select_key(unsigned score_bits) {
  if ((score_bits & 0x7FFFFFFFu) > 0x7F800000u) return kSelectNaN;
  if (score_bits == 0x80000000u) score_bits = 0;   // (zeros are equal)
  return score_bits & 0x80000000u ? ~score_bits : score_bits | 0x80000000u;
}

// ---- eviction ---------------------------------------------------------------------------------------------------------
// A list of kept tokens, ascending, moves to places 0, 1 .. of its sequence in chunks of `size`.  Who reads what a chunk writes: itself and the chunks before
// it, of which those have to have read that hold the tokens before the chunk's own that are kept from the places it writes.  before[i]: how many of the kept
// tokens are before place i * size (of places within the sequence).  At most two chunks: as many tokens, one behind the other in the list, as a chunk has.
struct EvictReaders {
  int first, count;   // chunks
};
IEX_HD EvictReaders evict_readers(int chunk, int size, int length, const int* before) {
  const int first = chunk * size, low = before[chunk], upto = length - first <= size ? first : before[chunk + 1], high = upto < first ? upto : first;
  return low < high ? EvictReaders{low / size, (high - 1) / size - low / size + 1} : EvictReaders{0, 0};
}
constexpr int kEvictAbandoned = -2;   // in the list, at the places of a chunk that gave up waiting

}  // namespace iex
