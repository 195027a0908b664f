// The plan of the document attention, on the host: which tiles of which document there are, longest work first.
// (As array expressions in Python this took 200 us for one short prompt, ten times its forward pass.)
#include <algorithm>
#include <vector>

#include "attention.cuh"

namespace ct {
namespace {

constexpr int64_t kKeyTile = 128, kGapTile = 64;
// A key tile's queries are all later tokens of the document, so the tiles' work differs by the document's length: tiles are
// cut into pieces of at most a quarter of an SM's share (2 and 3 leave the SMs uneven by up to 20 %, 6 and 8 write 1 to 2 %
// more shares than they even out; 4 x 4096 tokens, 32 heads), but not below 16 query tiles, whose work covers that of
// writing and adding a share.
constexpr int64_t kPiecesPerSm = 4, kSms = 148, kSmallestPiece = 16;

struct Document {
  int64_t start, length;
};

struct Piece {
  PlanRecord tile, range;
};

// Stable, by falling work; work is in [1, most].
template <typename T, typename Work> std::vector<T> sorted_by_work(const std::vector<T>& items, int64_t most, Work work) {
  std::vector<int64_t> place(static_cast<size_t>(most) + 2, 0);
  for (const T& item : items) ++place[most - work(item) + 1];
  for (size_t i = 1; i < place.size(); ++i) place[i] += place[i - 1];
  std::vector<T> sorted(items.size());
  for (const T& item : items) sorted[place[most - work(item)]++] = item;
  return sorted;
}

std::vector<PlanRecord> query_tiles(const std::vector<Document>& documents, int64_t step, int64_t longest) {
  std::vector<PlanRecord> tiles;
  for (const Document& d : documents)
    for (int64_t a = 0; a < d.length; a += step)
      tiles.push_back({static_cast<int>(d.start), static_cast<int>(d.length), static_cast<int>(a), 0});
  return sorted_by_work(tiles, longest, [&](const PlanRecord& r) { return std::min<int64_t>(r.length, r.a + step); });
}

int64_t build(const std::vector<Document>& documents, int64_t tokens, int heads, int kv_heads, int32_t* table, int64_t capacity,
              int64_t* sections, int64_t* key_slots) {
  int64_t longest = 1;
  for (const Document& d : documents) longest = std::max(longest, d.length);
  const int64_t tile_tokens = 128 / packed_heads(heads, kv_heads), head_blocks = heads / kv_heads / packed_heads(heads, kv_heads);
  std::vector<PlanRecord> parts[kPlanSections];
  parts[kPlanForward] = query_tiles(documents, 2 * tile_tokens, longest);
  parts[kPlanQuery] = query_tiles(documents, tile_tokens, longest);
  parts[kPlanTiles] = query_tiles(documents, kKeyTile, longest);

  auto work_of = [&](const Document& d, int64_t key) { return (d.length - key + tile_tokens - 1) / tile_tokens * head_blocks; };
  int64_t total = 0;
  for (const Document& d : documents)
    for (int64_t key = 0; key < d.length; key += kKeyTile) total += work_of(d, key);
  const int64_t largest = std::max(kSmallestPiece, (total * kv_heads + kSms * kPiecesPerSm - 1) / (kSms * kPiecesPerSm));
  std::vector<Piece> pieces;
  int64_t slots = 0;
  for (const Document& d : documents)
    for (int64_t key = 0; key < d.length; key += kKeyTile) {
      const int64_t work = work_of(d, key), count = (work + largest - 1) / largest;
      for (int64_t i = 0; i < count; ++i)
        pieces.push_back({{static_cast<int>(d.start), static_cast<int>(d.length), static_cast<int>(key), count > 1 ? static_cast<int>(slots + i) : -1},
                          {static_cast<int>(work * i / count), static_cast<int>(work * (i + 1) / count), 0, 0}});
      if (count > 1) {
        parts[kPlanReduce].push_back({static_cast<int>(d.start + key), static_cast<int>(std::min(kKeyTile, d.length - key)), static_cast<int>(slots),
                                      static_cast<int>(count)});
        slots += count;
      }
    }
  for (const Piece& p : sorted_by_work(pieces, largest, [](const Piece& p) { return static_cast<int64_t>(p.range.length) - p.range.start; })) {
    parts[kPlanKeys].push_back(p.tile);
    parts[kPlanKeys].push_back(p.range);
  }

  int64_t covered = 0;
  auto gap_until = [&](int64_t end) {
    for (; covered < end; covered += std::min(kGapTile, end - covered))
      parts[kPlanGaps].push_back({static_cast<int>(covered), static_cast<int>(std::min(kGapTile, end - covered)), 0, 0});
  };
  for (const Document& d : documents) {
    gap_until(d.start);
    covered = d.start + d.length;
  }
  gap_until(tokens);

  int64_t records = 0;
  for (int s = 0; s < kPlanSections; ++s) {
    sections[2 * s] = records;
    sections[2 * s + 1] = static_cast<int64_t>(parts[s].size()) / (s == kPlanKeys ? 2 : 1);
    if (table && records + static_cast<int64_t>(parts[s].size()) <= capacity)
      std::copy(parts[s].begin(), parts[s].end(), reinterpret_cast<PlanRecord*>(table) + records);
    records += static_cast<int64_t>(parts[s].size());
  }
  *key_slots = slots;
  return records;
}

}  // namespace
}  // namespace ct

using namespace ct;

extern "C" int64_t ct_attention_plan(const int64_t* starts, const int64_t* lengths, int64_t documents, int64_t tokens, int heads, int kv_heads,
                                     int32_t* table, int64_t capacity, int64_t* sections, int64_t* key_slots) {
  if (documents < 0 || tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || capacity < 0)
    return fail(CT_ERR_ARG, "ct_attention_plan: sizes");
  if (!sections || !key_slots || (documents && (!starts || !lengths))) return fail(CT_ERR_ARG, "ct_attention_plan: null pointer");
  if (tokens >= (int64_t(1) << 31) - 256) return fail(CT_ERR_UNSUPPORTED, "ct_attention_plan: %lld tokens", (long long)tokens);
  try {
    std::vector<Document> list;
    for (int64_t i = 0; i < documents; ++i) {
      if (lengths[i] < 0 || starts[i] < 0 || lengths[i] > tokens - starts[i])
        return fail(CT_ERR_ARG, "ct_attention_plan: document %lld lies outside the batch", (long long)i);
      if (lengths[i]) list.push_back({starts[i], lengths[i]});
    }
    std::stable_sort(list.begin(), list.end(), [](const Document& a, const Document& b) { return a.start < b.start; });
    for (size_t i = 1; i < list.size(); ++i)
      if (list[i].start < list[i - 1].start + list[i - 1].length) return fail(CT_ERR_ARG, "ct_attention_plan: document spans overlap");
    return build(list, tokens, heads, kv_heads, table, capacity, sections, key_slots);
  } catch (...) {                      // nothing is thrown across the boundary
    return fail(CT_ERR_ARG, "ct_attention_plan: out of host memory");
  }
}
