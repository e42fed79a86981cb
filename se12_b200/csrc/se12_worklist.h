// What a sequence adds to the attention kernels' work lists, in plain
// arithmetic (a test compiles it for the host). Lengths and row starts come
// from device memory and may hold anything: whatever they are, a sequence's
// rows lie in the batch's, its tokens in what its page table row can hold,
// and no sum leaves 31 bits.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define SE12_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define SE12_HOST_DEVICE inline
#endif

namespace se12 {

// A work list holds fewer units than this; a batch that counts more is not
// computed (the host refuses what its own sizes allow to get there).
constexpr long long kWorkLimit = (1ll << 31) - (1ll << 20);
// Positions a page table row may have.
constexpr int kMaxPositions = INT32_MAX - 4096;

SE12_HOST_DEVICE int int_min(int a, int b) { return a < b ? a : b; }
SE12_HOST_DEVICE int int_max(int a, int b) { return a > b ? a : b; }

// The batch's sizes, as the host knows them.
struct ListSizes {
  int tokens;    // rows of the token arrays
  int capacity;  // positions of a page table row, at most kMaxPositions
  int group;     // query rows per token and KV head
  int window;    // 0: none
};

// A sequence's rows and tokens.
struct SeqRows {
  int tokens;  // its rows
  int first;   // position of the first one (negative: inactive rows)
  int length;  // tokens in the cache that the page table can have
};

// Its first row in the token arrays.
SE12_HOST_DEVICE int first_row(int start, const ListSizes& z) { return int_min(int_max(start, 0), z.tokens); }

SE12_HOST_DEVICE SeqRows sequence_rows(int start, int stop, int len, const ListSizes& z) {
  SeqRows s;
  const int begin = first_row(start, z);
  s.tokens = int_min(int_max(stop, begin), z.tokens) - begin;
  s.length = int_max(len, 0);
  s.first = s.length - s.tokens;
  s.length = int_min(s.length, z.capacity);
  return s;
}

// The first position that a row at `pos` sees.
SE12_HOST_DEVICE int visible_from(int pos, int window) { return window ? int_max(int_max(pos, 0) - window + 1, 0) : 0; }

// Sums and products of units, up to the limit.
SE12_HOST_DEVICE int add_work(int a, int b, int limit) {  // each at most 2^31 - 1
  const unsigned sum = static_cast<unsigned>(a) + static_cast<unsigned>(b);
  return static_cast<int>(sum < static_cast<unsigned>(limit) ? sum : static_cast<unsigned>(limit));
}

SE12_HOST_DEVICE int times_work(int a, int b, int limit) {
  const long long product = static_cast<long long>(a) * b;
  return static_cast<int>(product < limit ? product : limit);
}

// A sequence's part of the list whose entries are chunks of tokens x row tiles.
struct SeqWork {
  SeqRows s;
  int low;     // first chunk's first token: a multiple of the chunk, at or below the first visible token
  int chunks;  // per pair (at least one: its CTA writes an empty sequence's zeros)
  int tiles;   // row tiles
};

SE12_HOST_DEVICE SeqWork sequence_work(const SeqRows& s, const ListSizes& z, int chunk, int rows) {
  SeqWork w;
  w.s = s;
  w.low = int_min(visible_from(s.first, z.window), s.length) / chunk * chunk;
  w.chunks = int_max((s.length - w.low + chunk - 1) / chunk, 1);
  w.tiles = (s.tokens * z.group + rows - 1) / rows;
  return w;
}

// A row tile's part of the list whose rows see different spans of tokens.
struct TileSpan {
  int low;      // first token, a multiple of the KV tile
  int chunks;   // KV tiles (at least one: its CTA writes the rows)
  int pos_min, pos_max;  // of its rows
};

// Past the last token of the span.
SE12_HOST_DEVICE int span_end(const SeqRows& s, int pos_max) { return pos_max < s.length ? pos_max + 1 : s.length; }

SE12_HOST_DEVICE TileSpan tile_span(const SeqRows& s, int tile, int tile_rows, const ListSizes& z, int kv_tile) {
  TileSpan p;
  p.pos_min = s.first + tile * tile_rows / z.group;
  p.pos_max = s.first + int_min(tile * tile_rows + tile_rows - 1, s.tokens * z.group - 1) / z.group;
  p.low = int_min(visible_from(p.pos_min, z.window), s.length) / kv_tile * kv_tile;
  p.chunks = int_max((span_end(s, p.pos_max) - p.low + kv_tile - 1) / kv_tile, 1);
  return p;
}

}  // namespace se12
