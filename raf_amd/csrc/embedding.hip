// Token embedding and its gradient for gfx950: `raf.op.embedding` / `raf.op.embedding_dx`
// (src/op/dialect/cuda/embedding.cc in the reference, which gathers and scatters unscaled rows).
//
// Forward: y[t] = scale * x[ids[t]], a gather that reads and writes each element once.
//
// Gradient: dx[r] = scale * sum over the tokens of row r of dy[t].  A sum by floating-point atomics
// would depend on the order in which they arrive, so tokens are sorted by row first:
//   1. tile_sort   sorts each tile of tokens by (row, position) in LDS;
//   2. row_sums    one wavefront per few rows looks its rows up in all sorted tiles at once (a
//                  binary search per lane and tile), writes zeros for rows without tokens, sums rows
//                  of up to kDirect tokens, and lists the others;
//   3. chunk_sums  sums the listed rows in chunks of kChunk tokens, a workgroup each, so that a
//                  token that fills half the batch is spread over the GPU;
//   4. chunk_join  adds the chunks of a row in order.
// Runs of a row are visited in tile order and sorted inside a tile, so every sum runs over
// ascending positions cut at multiples of kChunk: the result depends on the data alone although
// the list of long rows is filled in the order in which wavefronts arrive.  Up to kFewTokens
// tokens one launch does it all, every wavefront looking through all the ids.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "rafhip_vocab.h"
#include "status.h"
#include "vocab_io.h"

namespace rafhip {
namespace {

constexpr int kBlock = 256;
constexpr int kLanes = 64;
constexpr int kWaves = kBlock / kLanes;

// ------------------------------------------------------------------------------------- forward
template <typename TX, typename TY, typename Id>
__global__ __launch_bounds__(kBlock) void embedding_kernel(const TX* x, const Id* ids, int64_t n, int64_t rows,
                                                           int64_t first_row, int64_t width, int words,
                                                           int tokens_per_block, float scale, TY* y) {
  constexpr int kInFlight = 4;
  const int64_t t0 = (int64_t)blockIdx.x * tokens_per_block;
  const int tokens = (int)(n - t0 < tokens_per_block ? n - t0 : tokens_per_block);
  const unsigned items = (unsigned)tokens * (unsigned)words;
  for (unsigned i0 = threadIdx.x; i0 < items; i0 += kBlock * kInFlight) {
    typename Wide<TX>::Raw raw[kInFlight];
    int64_t to[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const unsigned i = i0 + u * kBlock;
      if (i < items) {
        const unsigned t = i / (unsigned)words, c = i - t * (unsigned)words;
        const uint64_t row = (uint64_t)(int64_t)ids[t0 + t] - (uint64_t)first_row;
        to[u] = (t0 + t) * width + (int64_t)c * kWide;
        if (row < (uint64_t)rows)
          raw[u] = Wide<TX>::load(x + (int64_t)row * width + (int64_t)c * kWide);
        else
          to[u] = ~to[u];  // no such row: zeros, whatever the scale
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (i0 + u * kBlock < items) {
        float v[kWide] = {};
        if (to[u] >= 0) {
#pragma unroll
          for (int j = 0; j < kWide; ++j) v[j] = scale * Wide<TX>::get(raw[u], j);
        }
        Wide<TY>::store(y + (to[u] >= 0 ? to[u] : ~to[u]), v);
      }
    }
  }
  const int rest = (int)(width - (int64_t)words * kWide);  // columns behind the last whole word
  const unsigned singles = (unsigned)tokens * (unsigned)rest;
  for (unsigned i = threadIdx.x; i < singles; i += kBlock) {
    const unsigned t = i / (unsigned)rest, c = i - t * (unsigned)rest;
    const uint64_t row = (uint64_t)(int64_t)ids[t0 + t] - (uint64_t)first_row;
    const int64_t col = (int64_t)words * kWide + c;
    const float v = row < (uint64_t)rows ? scale * Wide<TX>::one(x + (int64_t)row * width + col) : 0.f;
    Wide<TY>::put(y + (t0 + t) * width + col, v);
  }
}

// ------------------------------------------------------------------------------------ gradient
constexpr int kFewTokens = 256;  // one launch up to here
constexpr int kDirect = 32;      // tokens a wavefront sums by itself
constexpr int kChunk = 64;       // tokens of one partial sum of a longer row
constexpr int kPerWave = kChunk / kWaves;
constexpr int kMinTileBits = 11, kMaxTileBits = 14;
constexpr int kTilesPerRound = kLanes;  // a wavefront looks at this many tiles at once
constexpr int kMaxRounds = 8;
constexpr int kSortBlock = 1024;
constexpr int kInFlight = 8;  // token rows in flight per lane
constexpr uint32_t kNoToken = 0xffffffffu;

struct Layout {
  int tile_bits = 0;
  int tiles = 0;
  int64_t max_long = 0;   // rows of more than kDirect tokens
  int64_t max_items = 0;  // chunks of them
  int64_t max_parts = 0;  // chunks of rows with more than one
  int64_t keys_at = 0, counters_at = 0, rows_at = 0, items_at = 0, runs_at = 0, parts_at = 0, bytes = 0;
};

// A row of more than kDirect tokens: where its runs are listed and what it is cut into.
struct LongRow {
  uint32_t row, tokens, n_runs, first_run, first_part;
};
struct Item {
  uint32_t long_row, chunk;
};
struct Run {
  uint32_t at, before;  // first key of the run; tokens of the row in earlier runs
};
enum { kLongRows = 0, kItems, kRuns, kParts, kCounters };

inline int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// False if the sizes are not supported.
bool layout_of(int64_t n, int64_t rows, int64_t width, Layout* l) {
  if (rows >= (1LL << 21)) return false;
  int row_bits = 1;  // the largest key stays free for "no token"
  while ((1LL << row_bits) <= rows) ++row_bits;
  const int most = 32 - row_bits < kMaxTileBits ? 32 - row_bits : kMaxTileBits;
  int bits = kMinTileBits;
  while (bits < most && (n >> bits) >= kTilesPerRound) ++bits;
  const int64_t tiles = (n + (1LL << bits) - 1) >> bits;
  if (tiles > kTilesPerRound * kMaxRounds) return false;
  l->tile_bits = bits;
  l->tiles = (int)tiles;
  l->max_long = n / (kDirect + 1);
  l->max_parts = n / kChunk + n / (kChunk + 1);
  l->max_items = n / kChunk + l->max_long;
  auto take = [&](int64_t bytes) {
    const int64_t at = l->bytes;
    l->bytes += align256(bytes);
    return at;
  };
  l->counters_at = take(kCounters * 4);
  l->keys_at = take((tiles << bits) * 4);
  l->rows_at = take(l->max_long * (int64_t)sizeof(LongRow));
  l->items_at = take(l->max_items * (int64_t)sizeof(Item));
  l->runs_at = take((n < l->max_long * tiles ? n : l->max_long * tiles) * (int64_t)sizeof(Run));
  l->parts_at = take(l->max_parts * width * 4);
  return true;
}

// The row a token belongs to, or -1.
struct Which {
  int64_t rows, first_row, padding;
  int has_padding;
  __device__ __forceinline__ int64_t row(int64_t id) const {
    const uint64_t r = (uint64_t)id - (uint64_t)first_row;
    return r < (uint64_t)rows && !(has_padding && id == padding) ? (int64_t)r : -1;
  }
};

// Sorts one tile in LDS by a bitonic network over (row << tile_bits | position).
template <typename Id>
__global__ __launch_bounds__(kSortBlock) void tile_sort(const Id* ids, int64_t n, Which which, int tile_bits,
                                                        uint32_t* keys, uint32_t* counters) {
  extern __shared__ uint32_t tile[];
  const int size = 1 << tile_bits;
  const int64_t t0 = (int64_t)blockIdx.x << tile_bits;
  if (blockIdx.x == 0 && threadIdx.x < kCounters) counters[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < size; i += kSortBlock) {
    const int64_t row = t0 + i < n ? which.row((int64_t)ids[t0 + i]) : -1;
    tile[i] = row >= 0 ? (uint32_t)row << tile_bits | (uint32_t)i : kNoToken;
  }
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kSortBlock) {
        const int a = (i & (j - 1)) | (i & ~(j - 1)) << 1, b = a | j;
        const uint32_t x = tile[a], y = tile[b];
        const bool up = (a & k) == 0;
        if ((x > y) == up) {
          tile[a] = y;
          tile[b] = x;
        }
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < size; i += kSortBlock) keys[t0 + i] = tile[i];
}

// First index in a sorted tile whose key is not below `key`.
__device__ __forceinline__ int lower_bound(const uint32_t* tile, int size, uint32_t key) {
  int at = 0;
  for (int step = size >> 1; step > 0; step >>= 1)
    if (tile[at + step - 1] < key) at += step;
  return at + (tile[at] < key ? 1 : 0);
}

// Columns [col, col + kCols) of the sum over `count` tokens, of which lane e of `token` holds the
// e-th; lanes that are not active have no column.  `count` is the same in all lanes.
template <typename TD, int kCols>
__device__ __forceinline__ void add_tokens(const TD* dy, int64_t width, int64_t col, bool active, int token, int first,
                                           int count, float (&acc)[kCols]) {
  for (int e0 = 0; e0 < count; e0 += kInFlight) {
    if constexpr (kCols == kWide) {
      typename Wide<TD>::Raw raw[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        if (e0 + u < count) {
          const int64_t t = __builtin_amdgcn_readlane(token, first + e0 + u);
          if (active) raw[u] = Wide<TD>::load(dy + t * width + col);
        }
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        if (e0 + u < count && active) {
#pragma unroll
          for (int j = 0; j < kWide; ++j) acc[j] += Wide<TD>::get(raw[u], j);
        }
      }
    } else {
      float one[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        if (e0 + u < count) {
          const int64_t t = __builtin_amdgcn_readlane(token, first + e0 + u);
          if (active) one[u] = Wide<TD>::one(dy + t * width + col);
        }
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (e0 + u < count && active) acc[0] += one[u];
    }
  }
}

// dx = [dx +] scale * acc.
template <typename TO, int kCols>
__device__ __forceinline__ void put_row(TO* at, const float (&acc)[kCols], float scale, bool accumulate) {
  float v[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) v[j] = scale * acc[j];
  if constexpr (kCols == kWide) {
    if (accumulate) {
      const typename Wide<TO>::Raw old = Wide<TO>::load(at);
#pragma unroll
      for (int j = 0; j < kWide; ++j) v[j] += Wide<TO>::get(old, j);
    }
    Wide<TO>::store(at, v);
  } else {
    if (accumulate) v[0] += Wide<TO>::one(at);
    Wide<TO>::put(at, v[0]);
  }
}

// Calls f(col, active, whole word or single column) so that the wavefront covers `width` columns.
template <typename F>
__device__ __forceinline__ void for_columns(int64_t width, F&& f) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t words = width / kWide;
  for (int64_t w = 0; w < words; w += kLanes) f(std::integral_constant<int, kWide>{}, (w + lane) * kWide, w + lane < words);
  const int64_t rest = words * kWide;
  if (rest < width) f(std::integral_constant<int, 1>{}, rest + lane, rest + lane < width);
}

template <typename TO>
__device__ __forceinline__ void zero_row(TO* at, int64_t width) {
  for_columns(width, [&](auto cols, int64_t col, bool active) {
    const float none[decltype(cols)::value] = {};
    if (active) put_row<TO, decltype(cols)::value>(at + col, none, 0.f, false);
  });
}

// One row whose tokens (at most kLanes) the lanes hold.
template <typename TD, typename TO>
__device__ __forceinline__ void sum_row(const TD* dy, int64_t width, int token, int count, float scale, bool accumulate,
                                        TO* at) {
  for_columns(width, [&](auto cols, int64_t col, bool active) {
    float acc[decltype(cols)::value] = {};
    add_tokens<TD, decltype(cols)::value>(dy, width, col, active, token, 0, count, acc);
    if (active) put_row<TO, decltype(cols)::value>(at + col, acc, scale, accumulate);
  });
}

// All of the gradient for up to kFewTokens tokens: every wavefront looks through the ids for its rows.
template <typename TD, typename TO, typename Id>
__global__ __launch_bounds__(kBlock) void few_tokens(const TD* dy, const Id* ids, int n, Which which, int64_t width,
                                                     float scale, int accumulate, int rows_per_wave, TO* dx) {
  constexpr int kRounds = kFewTokens / kLanes;
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t r0 = wave * rows_per_wave;
  if (r0 >= which.rows) return;
  const int mine = (int)(which.rows - r0 < rows_per_wave ? which.rows - r0 : rows_per_wave);
  int64_t row[kRounds];
  bool any = false;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int t = k * kLanes + lane;
    row[k] = t < n ? which.row((int64_t)ids[t]) - r0 : -1;
    any |= row[k] >= 0 && row[k] < mine;
  }
  const bool some = __any(any);
  for (int i = 0; i < mine; ++i) {
    TO* at = dx + (r0 + i) * width;
    uint64_t hits[kRounds] = {};
    uint64_t all = 0;
    if (some) {
#pragma unroll
      for (int k = 0; k < kRounds; ++k) all |= hits[k] = __ballot(row[k] == i);
    }
    if (all == 0) {
      if (!accumulate) zero_row(at, width);
      continue;
    }
    for_columns(width, [&](auto cols, int64_t col, bool active) {
      constexpr int kCols = decltype(cols)::value;
      float acc[kCols] = {};
#pragma unroll
      for (int k = 0; k < kRounds; ++k) {
        // The set bits in ascending order: lane e learns the position of the e-th.
        const uint64_t m = hits[k];
        const int count = __popcll(m);
        if (count == 0) continue;
        const bool set = m >> lane & 1;
        const int place = __popcll(m & ((1ull << lane) - 1));
        // A lane that holds a token sends it to the lane of its rank, the others behind the last.
        const int token = __builtin_amdgcn_ds_permute((set ? place : count + (lane - place)) * 4, k * kLanes + lane);
        add_tokens<TD, kCols>(dy, width, col, active, token, 0, count, acc);
      }
      if (active) put_row<TO, kCols>(at + col, acc, scale, accumulate != 0);
    });
  }
}

// Rows of a wavefront: kGroup rows side by side, `spread` lanes (one per tile) each; with more
// than 64 tiles one row at a time in kRounds rounds.
template <typename TD, typename TO, int kRounds>
__global__ __launch_bounds__(kBlock) void row_sums(const TD* dy, const uint32_t* keys, int tiles, int tile_bits,
                                                   int spread_bits, int group, int64_t rows, int64_t width, float scale,
                                                   int accumulate, TO* dx, uint32_t* counters, LongRow* long_rows,
                                                   Item* items, Run* runs) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t n_waves = (int64_t)gridDim.x * kWaves;
  const int size = 1 << tile_bits;
  const int spread = 1 << spread_bits;
  const int slot = lane >> spread_bits, tile0 = lane & (spread - 1);
  for (int64_t r0 = wave * group; r0 < rows; r0 += n_waves * group) {
    const int64_t my_row = r0 + slot;
    uint32_t at[kRounds];
    int len[kRounds], before[kRounds];
    int total = 0;  // tokens of this lane's row, the same in all its lanes
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      const int t = q * kTilesPerRound + tile0;
      at[q] = 0;
      len[q] = 0;
      if (slot < group && my_row < rows && t < tiles) {
        const uint32_t* tile = keys + ((int64_t)t << tile_bits);
        const int lo = lower_bound(tile, size, (uint32_t)my_row << tile_bits);
        const int hi = lower_bound(tile, size, (uint32_t)(my_row + 1) << tile_bits);
        at[q] = ((uint32_t)t << tile_bits) + (uint32_t)lo;
        len[q] = hi - lo;
      }
      int sum = len[q];  // inclusive over the row's lanes
      for (int d = 1; d < spread; d <<= 1) {
        const int up = __shfl_up(sum, d, spread);
        if (tile0 >= d) sum += up;
      }
      before[q] = total + sum - len[q];
      total += __shfl(sum, spread - 1, spread);
    }
    const int here = (int)(rows - r0 < group ? rows - r0 : group);
    for (int i = 0; i < here; ++i) {
      TO* out = dx + (r0 + i) * width;
      const int count = __builtin_amdgcn_readlane(total, i << spread_bits);
      if (count == 0) {
        if (!accumulate) zero_row(out, width);
        continue;
      }
      if (count <= kDirect) {
        int key_at = 0;  // lane e: where the e-th token's key is
#pragma unroll
        for (int q = 0; q < kRounds; ++q) {
          uint64_t some = __ballot(slot == i && len[q] > 0);
          while (some) {
            const int src = __ffsll((unsigned long long)some) - 1;
            some &= some - 1;
            const int a = __builtin_amdgcn_readlane((int)at[q], src), b = __builtin_amdgcn_readlane(before[q], src);
            if (lane >= b) key_at = a + (lane - b);
          }
        }
        int token = 0;
        if (lane < count) {
          const uint32_t tile = (uint32_t)key_at >> tile_bits;
          token = (int)((tile << tile_bits) + (keys[key_at] & (uint32_t)(size - 1)));
        }
        sum_row(dy, width, token, count, scale, accumulate != 0, out);
        continue;
      }
      // Listed for the next launch.
      int n_runs = 0;
      int place[kRounds];
#pragma unroll
      for (int q = 0; q < kRounds; ++q) {
        const uint64_t some = __ballot(slot == i && len[q] > 0);
        place[q] = n_runs + __popcll(some & ((1ull << lane) - 1));
        n_runs += __popcll(some);
      }
      const int chunks = (count + kChunk - 1) / kChunk;
      uint32_t base = 0;
      if (lane < kCounters)
        base = atomicAdd(&counters[lane], (uint32_t)(lane == kLongRows ? 1 : lane == kItems ? chunks : lane == kRuns ? n_runs : chunks > 1 ? chunks : 0));
      const uint32_t id = __builtin_amdgcn_readlane((int)base, kLongRows);
      const uint32_t first_item = __builtin_amdgcn_readlane((int)base, kItems);
      const uint32_t first_run = __builtin_amdgcn_readlane((int)base, kRuns);
      if (lane == 0) {
        const uint32_t first_part = __builtin_amdgcn_readlane((int)base, kParts);
        long_rows[id] = LongRow{(uint32_t)(r0 + i), (uint32_t)count, (uint32_t)n_runs, first_run, first_part};
      }
      for (int c = lane; c < chunks; c += kLanes) items[first_item + c] = Item{id, (uint32_t)c};
#pragma unroll
      for (int q = 0; q < kRounds; ++q)
        if (slot == i && len[q] > 0) runs[first_run + place[q]] = Run{at[q], (uint32_t)before[q]};
    }
  }
}

// One chunk of a long row per workgroup: each wavefront sums kPerWave tokens, the four sums are
// added in order, and the result is the row (a row of one chunk) or a partial sum.
template <typename TD, typename TO>
__global__ __launch_bounds__(kBlock) void chunk_sums(const TD* dy, const uint32_t* keys, int tile_bits, int64_t width,
                                                     float scale, int accumulate, TO* dx, const uint32_t* counters,
                                                     const LongRow* long_rows, const Item* items, const Run* runs,
                                                     float* parts) {
  __shared__ float sums[kWaves][kLanes * kWide];
  const int lane = threadIdx.x & (kLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const uint32_t n_items = counters[kItems];
  for (uint32_t it = blockIdx.x; it < n_items; it += gridDim.x) {
    const Item item = items[it];
    const LongRow row = long_rows[item.long_row];
    const int first = (int)item.chunk * kChunk + wave * kPerWave;
    int count = (int)row.tokens - first;
    count = count < 0 ? 0 : count > kPerWave ? kPerWave : count;
    int token = 0;
    if (lane < count) {  // the run that holds this lane's token
      const Run* r = runs + row.first_run;
      const uint32_t want = (uint32_t)(first + lane);
      uint32_t lo = 0, hi = row.n_runs;  // the last run that starts at or before it
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (r[mid].before <= want)
          lo = mid;
        else
          hi = mid;
      }
      const uint32_t key_at = r[lo].at + (want - r[lo].before);
      token = (int)((key_at >> tile_bits << tile_bits) + (keys[key_at] & ((1u << tile_bits) - 1)));
    }
    const bool whole = row.tokens <= (uint32_t)kChunk;
    for_columns(width, [&](auto cols, int64_t col, bool active) {
      constexpr int kCols = decltype(cols)::value;
      float acc[kCols] = {};
      add_tokens<TD, kCols>(dy, width, col, active, token, 0, count, acc);
      __syncthreads();  // the sums of the previous columns have been read
#pragma unroll
      for (int j = 0; j < kCols; ++j) sums[wave][lane * kCols + j] = acc[j];
      __syncthreads();
      const int64_t c0 = col - (int64_t)lane * kCols;  // the first column of lane 0
      const int64_t end = kCols == kWide ? width / kWide * kWide : width;
      for (int c = threadIdx.x; c < kLanes * kCols && c0 + c < end; c += kBlock) {
        float total[1] = {((sums[0][c] + sums[1][c]) + sums[2][c]) + sums[3][c]};
        if (whole)
          put_row<TO, 1>(dx + (int64_t)row.row * width + c0 + c, total, scale, accumulate != 0);
        else
          parts[((int64_t)row.first_part + item.chunk) * width + c0 + c] = total[0];
      }
    });
  }
}

// The chunks of a long row added in order: 64 columns per workgroup, four stretches of chunks.
template <typename TO>
__global__ __launch_bounds__(kBlock) void chunk_join(int64_t width, float scale, int accumulate, TO* dx,
                                                     const uint32_t* counters, const LongRow* long_rows,
                                                     const float* parts) {
  __shared__ float sums[kWaves][kLanes];
  const int lane = threadIdx.x & (kLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t col = (int64_t)blockIdx.x * kLanes + lane;
  const uint32_t n_long = counters[kLongRows];
  for (uint32_t h = blockIdx.y; h < n_long; h += gridDim.y) {
    const LongRow row = long_rows[h];
    if (row.tokens <= (uint32_t)kChunk) continue;
    const int chunks = (int)((row.tokens + kChunk - 1) / kChunk);
    const int per = (chunks + kWaves - 1) / kWaves;
    const int from = wave * per, to = from + per < chunks ? from + per : chunks;
    float acc = 0.f;
    if (col < width) {
      const float* p = parts + (int64_t)row.first_part * width + col;
      for (int c0 = from; c0 < to; c0 += kInFlight) {
        float v[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u)
          if (c0 + u < to) v[u] = p[(int64_t)(c0 + u) * width];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u)
          if (c0 + u < to) acc += v[u];
      }
    }
    __syncthreads();
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && col < width) {
      float total[1] = {((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane]};
      put_row<TO, 1>(dx + (int64_t)row.row * width + col, total, scale, accumulate != 0);
    }
  }
}

constexpr int kFewRowsPerWave = 8;
constexpr int64_t kMaxRowBlocks = 2048;   // workgroups of row_sums: eight per CU, each strides over rows
constexpr int64_t kMaxChunkBlocks = 2048;

template <typename TD, typename TO, typename Id>
void launch_dx(const TD* dy, const Id* ids, int64_t n, const Which& which, int64_t width, float scale, int accumulate,
               TO* dx, char* ws, const Layout& l, hipStream_t s) {
  const int64_t rows = which.rows;
  if (n <= kFewTokens) {
    const int64_t waves = (rows + kFewRowsPerWave - 1) / kFewRowsPerWave;
    hipLaunchKernelGGL((few_tokens<TD, TO, Id>), dim3((unsigned)((waves + kWaves - 1) / kWaves)), dim3(kBlock), 0, s, dy, ids,
                       (int)n, which, width, scale, accumulate, kFewRowsPerWave, dx);
    return;
  }
  auto* counters = reinterpret_cast<uint32_t*>(ws + l.counters_at);
  auto* keys = reinterpret_cast<uint32_t*>(ws + l.keys_at);
  auto* long_rows = reinterpret_cast<LongRow*>(ws + l.rows_at);
  auto* items = reinterpret_cast<Item*>(ws + l.items_at);
  auto* runs = reinterpret_cast<Run*>(ws + l.runs_at);
  auto* parts = reinterpret_cast<float*>(ws + l.parts_at);
  hipLaunchKernelGGL(tile_sort<Id>, dim3((unsigned)l.tiles), dim3(kSortBlock), (size_t)4 << l.tile_bits, s, ids, n, which,
                     l.tile_bits, keys, counters);
  int spread_bits = 0;
  while (spread_bits < 6 && (1 << spread_bits) < l.tiles) ++spread_bits;
  int group = kLanes >> spread_bits;
  if (group > kFewRowsPerWave) group = kFewRowsPerWave;
  const int64_t waves = (rows + group - 1) / group;
  int64_t blocks = (waves + kWaves - 1) / kWaves;
  if (blocks > kMaxRowBlocks) blocks = kMaxRowBlocks;
  auto rows_go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, s, dy, keys, l.tiles, l.tile_bits, spread_bits,
                       group, rows, width, scale, accumulate, dx, counters, long_rows, items, runs);
  };
  l.tiles <= kTilesPerRound ? rows_go(row_sums<TD, TO, 1>) : rows_go(row_sums<TD, TO, kMaxRounds>);
  const int64_t chunk_blocks = l.max_items < kMaxChunkBlocks ? l.max_items : kMaxChunkBlocks;
  hipLaunchKernelGGL((chunk_sums<TD, TO>), dim3((unsigned)chunk_blocks), dim3(kBlock), 0, s, dy, keys, l.tile_bits, width,
                     scale, accumulate, dx, counters, long_rows, items, runs, parts);
  const int64_t most = n / (kChunk + 1);
  hipLaunchKernelGGL(chunk_join<TO>, dim3((unsigned)((width + kLanes - 1) / kLanes), (unsigned)(most < 64 ? most : 64)),
                     dim3(kBlock), 0, s, width, scale, accumulate, dx, counters, long_rows, parts);
}

int check_common(const char* who, int32_t a_dtype, int32_t b_dtype, int64_t rows, int64_t width, int32_t index_bits, int64_t n,
                 int64_t first_row) {
  if (element_bytes(a_dtype) == 0 || element_bytes(b_dtype) == 0)
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: dtypes %d and %d", who, a_dtype, b_dtype);
  if (index_bits != 32 && index_bits != 64) return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %d-bit indices", who, index_bits);
  if (n < 0 || rows < 0 || width < 0)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: n = %lld, rows = %lld, width = %lld", who, (long long)n, (long long)rows, (long long)width);
  if (first_row < 0 || first_row > INT64_MAX - rows)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: first_row = %lld", who, (long long)first_row);
  // Byte offsets stay far inside 63 bits, and the column arithmetic of a workgroup inside 31.
  if (width >= (1LL << 24) || rows >= (1LL << 36) || n >= (1LL << 36))
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %lld rows, %lld tokens of width %lld", who, (long long)rows, (long long)n, (long long)width);
  return RAFHIP_OK;
}

}  // namespace
}  // namespace rafhip

extern "C" int rafhip_embedding(const void* x, int32_t x_dtype, int64_t rows, int64_t width, const void* indices,
                                int32_t index_bits, int64_t n, int64_t first_row, float scale, void* y, int32_t y_dtype,
                                void* stream) {
  using namespace rafhip;
  clear_error();
  const char* who = "rafhip_embedding";
  if (int st = check_common(who, x_dtype, y_dtype, rows, width, index_bits, n, first_row)) return st;
  if (n == 0 || width == 0) return RAFHIP_OK;
  if ((rows > 0 && !x) || !indices || !y) return fail(RAFHIP_ERR_INVALID_ARG, "%s: null tensor", who);
  if (!is_aligned(x, element_bytes(x_dtype)) || !is_aligned(y, element_bytes(y_dtype)) || !is_aligned(indices, index_bits / 8))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  const int words = (int)(width / kWide);
  // Four words in flight per lane where that still leaves every CU several workgroups, one where it does not.
  const int64_t all = n * (words > 0 ? words : 1);
  const int64_t per_block = all >= 256 * 8 * 4 * (int64_t)kBlock ? 4 * kBlock : kBlock;
  int64_t tokens = per_block / (words > 0 ? words : 1);
  tokens = tokens < 1 ? 1 : tokens;
  const int64_t blocks = (n + tokens - 1) / tokens;
  if (blocks > INT32_MAX) return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %lld tokens", who, (long long)n);
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_element(x_dtype, [&](auto tx) {
    with_element(y_dtype, [&](auto ty) {
      with_index(index_bits, [&](auto id) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        using Id = decltype(id);
        hipLaunchKernelGGL((embedding_kernel<TX, TY, Id>), dim3((unsigned)blocks), dim3(kBlock), 0, s,
                           static_cast<const TX*>(x), static_cast<const Id*>(indices), n, rows, first_row, width, words,
                           (int)tokens, scale, static_cast<TY*>(y));
      });
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}

extern "C" int64_t rafhip_embedding_dx_workspace_bytes(int64_t n, int64_t rows, int64_t width) {
  using namespace rafhip;
  if (n < 0 || rows < 0 || width < 0 || width >= (1LL << 24)) return -1;
  Layout l;
  if (!layout_of(n, rows, width, &l)) return -1;
  return n <= kFewTokens || rows == 0 || width == 0 ? 0 : l.bytes;
}

extern "C" int rafhip_embedding_dx(const void* dy, int32_t dy_dtype, const void* indices, int32_t index_bits, int64_t n,
                                   int64_t rows, int64_t width, int64_t first_row, int32_t has_padding,
                                   int64_t padding_index, float scale, void* dx, int32_t dx_dtype, int32_t accumulate,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace rafhip;
  clear_error();
  const char* who = "rafhip_embedding_dx";
  if (int st = check_common(who, dy_dtype, dx_dtype, rows, width, index_bits, n, first_row)) return st;
  const int64_t need = rafhip_embedding_dx_workspace_bytes(n, rows, width);
  if (need < 0)
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %lld tokens over %lld rows", who, (long long)n, (long long)rows);
  if (rows == 0 || width == 0) return RAFHIP_OK;
  if (!dx || (n > 0 && (!dy || !indices))) return fail(RAFHIP_ERR_INVALID_ARG, "%s: null tensor", who);
  if (!is_aligned(dy, element_bytes(dy_dtype)) || !is_aligned(dx, element_bytes(dx_dtype)) || !is_aligned(indices, index_bits / 8))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p of %lld bytes, need %lld", who, workspace, (long long)workspace_bytes,
                (long long)need);
  if (need > 0 && !is_aligned(workspace, 16)) return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p is not 16-byte aligned", who, workspace);
  if (n == 0 && accumulate) return RAFHIP_OK;
  Layout l;
  layout_of(n, rows, width, &l);
  const Which which{rows, first_row, padding_index, has_padding != 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_element(dy_dtype, [&](auto td) {
    with_element(dx_dtype, [&](auto to) {
      with_index(index_bits, [&](auto id) {
        using TD = decltype(td);
        using TO = decltype(to);
        using Id = decltype(id);
        launch_dx(static_cast<const TD*>(dy), static_cast<const Id*>(indices), n, which, width, scale, accumulate != 0,
                  static_cast<TO*>(dx), static_cast<char*>(workspace), l, s);
      });
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}
