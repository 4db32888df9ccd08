// Token embedding and its gradient for gfx950: `raf.op.embedding` / `raf.op.embedding_dx`
// (src/op/dialect/cuda/embedding.cc in the reference, which gathers and scatters unscaled rows).
//
// Forward: y[t] = scale * x[ids[t]], a gather that reads and writes each element once.
//
// Gradient: dx[r] = scale * sum over the tokens of row r of dy[t].  A sum by floating-point atomics
// would depend on the order in which they arrive, so tokens are sorted by row first:
//   1. tile_sort   sorts each tile of tokens by (row, position);
//   2. find_rows   looks every row up in all sorted tiles at once (a binary search per lane and
//                  tile), writes zeros for rows without tokens, and lists the others: the tokens of
//                  rows of up to kDirect, and chunks of kChunk tokens of longer rows;
//   3. sum_rows    sums what is listed, a chunk per workgroup and the short rows by wavefronts, so
//                  that a token that fills half the batch is spread over the GPU;
//   4. join_chunks adds the chunks of a row in order.
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
constexpr int kDirect = 8;       // tokens of a row that one wavefront sums
constexpr int kChunk = 64;       // tokens of one partial sum of a longer row
constexpr int kChunkBlock = 512;
constexpr int kChunkWaves = kChunkBlock / kLanes;
constexpr int kPerWave = kChunk / kChunkWaves;
constexpr int kMinTileBits = 11, kMaxTileBits = 14;
constexpr int kMaxTiles = 512;
constexpr int kGroup = kLanes / kDirect;  // rows of a wavefront: their tokens have a lane each
constexpr int kSortBlock = 1024;
constexpr int kInFlight = 8;  // words in flight per lane
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr int kSlotShift = 28;  // an entry: a token (23 bits: kMaxTiles tiles of 2^14) and its row's slot

struct Layout {
  int tile_bits = 0;
  int tiles = 0;
  int bucket_bits = 0;  // log2 of the rows that share an entry of a tile's index
  int buckets = 0;
  int64_t max_singles = 0;  // rows of more than kDirect tokens and no more than a chunk
  int64_t max_runs = 0;   // runs of them
  int64_t max_parts = 0;  // chunks of rows with more than one
  int64_t keys_at = 0, index_at = 0, taken_at = 0, entries_at = 0, counts_at = 0, singles_at = 0, items_at = 0, runs_at = 0, parts_at = 0, bytes = 0;
};

// One chunk of a row of more than kDirect tokens, with all that its sum needs to know.  There are two
// lists: rows of one chunk, and the chunks of the others, whose place there is that of their
// partial sum.
struct Item {
  uint32_t row, tokens, n_runs, first_run, chunk;
};
struct Run {
  uint32_t at, before;  // first key of the run; tokens of the row in earlier runs
};
// How much of each list is taken, in one word: a wavefront reserves all it needs with one atomic
// (with four, 800 wavefronts queued for some 60 us).
typedef unsigned long long Taken;
constexpr int kRunBits = 24, kSingleBits = 21;  // up to 2^23 runs, 2^20 rows of one chunk, 2^18 chunks
__device__ __forceinline__ Taken take(uint32_t runs, uint32_t chunks) {
  return (Taken)runs | (chunks == 1 ? (Taken)1 << kRunBits : (Taken)chunks << (kRunBits + kSingleBits));
}
__device__ __forceinline__ uint32_t runs_of(Taken t) { return (uint32_t)t & ((1u << kRunBits) - 1); }
__device__ __forceinline__ uint32_t singles_of(Taken t) { return (uint32_t)(t >> kRunBits) & ((1u << kSingleBits) - 1); }
__device__ __forceinline__ uint32_t parts_of(Taken t) { return (uint32_t)(t >> (kRunBits + kSingleBits)); }

inline int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// False if the sizes are not supported.
bool layout_of(int64_t n, int64_t rows, int64_t width, Layout* l) {
  if (rows >= (1LL << 21)) return false;
  int row_bits = 1;  // the largest key stays free for "no token"
  while ((1LL << row_bits) <= rows) ++row_bits;
  const int most = 32 - row_bits < kMaxTileBits ? 32 - row_bits : kMaxTileBits;
  int bits = kMinTileBits;
  while (bits < most && (n >> bits) >= kLanes) ++bits;
  const int64_t tiles = (n + (1LL << bits) - 1) >> bits;
  if (tiles > kMaxTiles) return false;
  l->tile_bits = bits;
  l->tiles = (int)tiles;
  // r rows of n tokens together have at most n / kChunk + r chunks.
  const int64_t listed = n / (kDirect + 1);
  l->max_singles = listed;
  l->max_runs = n < listed * tiles ? n : listed * tiles;
  l->max_parts = n / kChunk + n / (kChunk + 1);
  auto place = [&](int64_t bytes) {
    const int64_t at = l->bytes;
    l->bytes += align256(bytes);
    return at;
  };
  l->taken_at = place(sizeof(Taken));
  l->keys_at = place((tiles << bits) * 4);
  // About one key per entry, or 16 rows where the keys are many: a search then takes a step or two.
  int bucket = row_bits - bits;
  if (bucket < 4) bucket = 4;
  l->bucket_bits = bucket;
  l->buckets = (int)((rows + (1LL << bucket) - 1) >> bucket);
  l->index_at = place(tiles * (l->buckets + 1) * 2);
  l->entries_at = place((rows + kGroup) * kDirect * 4);
  l->counts_at = place(rows * 4);
  l->singles_at = place(l->max_singles * (int64_t)sizeof(Item));
  l->items_at = place(l->max_parts * (int64_t)sizeof(Item));
  l->runs_at = place(l->max_runs * (int64_t)sizeof(Run));
  l->parts_at = place(l->max_parts * width * 4);
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

// Sorts one tile by a bitonic network over (row << tile_bits | position), kEach = 2^tile_bits /
// kSortBlock keys in the registers of each thread: key i sits in register i % kEach of thread
// i / kEach, so of the 66 stages of 2048 keys 11 stay inside a thread, 45 inside a wavefront and 10
// go through LDS.  Then the index: for every bucket of rows the first key that is not below it.
template <typename Id, int kEach>
__global__ __launch_bounds__(kSortBlock) void tile_sort(const Id* ids, int64_t n, Which which, int tile_bits,
                                                        int bucket_bits, int buckets, uint32_t* keys, uint16_t* index,
                                                        Taken* taken) {
  constexpr int kSize = kEach * kSortBlock;
  __shared__ uint32_t lds[kSize];
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * kSize;
  if (blockIdx.x == 0 && tid == 0) *taken = 0;
  uint32_t v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kSortBlock + tid;  // any order will do before the sort
    const int64_t row = t0 + i < n ? which.row((int64_t)ids[t0 + i]) : -1;
    v[e] = row >= 0 ? (uint32_t)row << tile_bits | (uint32_t)i : kNoToken;
  }
#pragma unroll 1
  for (int k = 2; k <= kSize; k <<= 1) {
    for (int j = k >> 1; j >= kEach * kLanes; j >>= 1) {  // across wavefronts
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) lds[e * kSortBlock + tid] = v[e];
      __syncthreads();
      const int other = tid ^ (j / kEach);
      const bool low = (tid & (j / kEach)) == 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const uint32_t y = lds[e * kSortBlock + other];
        const bool up = ((tid * kEach + e) & k) == 0;
        v[e] = low == up ? min(v[e], y) : max(v[e], y);
      }
    }
    for (int j = (k >> 1) < kEach * kLanes ? k >> 1 : kEach * kLanes / 2; j >= kEach; j >>= 1) {  // across lanes
      const bool low = (tid & (j / kEach)) == 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const uint32_t y = __shfl_xor(v[e], j / kEach, kLanes);
        const bool up = ((tid * kEach + e) & k) == 0;
        v[e] = low == up ? min(v[e], y) : max(v[e], y);
      }
    }
#pragma unroll
    for (int j = kEach / 2; j > 0; j >>= 1) {  // across registers
      if (j >= k) continue;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (e & j) continue;
        const bool up = ((tid * kEach + e) & k) == 0;
        const uint32_t x = v[e], y = v[e | j];
        v[e] = up ? min(x, y) : max(x, y);
        v[e | j] = up ? max(x, y) : min(x, y);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) lds[tid * kEach + e] = v[e];
  __syncthreads();
  for (int i = tid; i < kSize; i += kSortBlock) keys[t0 + i] = lds[i];
  for (int b = tid; b <= buckets; b += kSortBlock) {
    // The last entry lies behind every row; its key may exceed 32 bits.
    const uint64_t key = (uint64_t)b << (bucket_bits + tile_bits);
    int at = 0;
    for (int step = kSize >> 1; step > 0; step >>= 1)
      if (lds[at + step - 1] < key) at += step;
    at += lds[at] < key ? 1 : 0;
    index[(int64_t)blockIdx.x * (buckets + 1) + b] = (uint16_t)at;
  }
}

// A wavefront's share of a row: kSweeps words per lane, 64 words apart, or single columns.
// Adds `count` tokens, of which lane first + e of `token` holds the e-th; `count` is the same in all
// lanes.  kInFlight words are requested before the first is needed: of several tokens, or of one token
// where rows are long and tokens few.
template <typename TD, int kSweeps>
__device__ __forceinline__ void add_words(const TD* dy, int64_t width, int64_t word, int64_t words, int token, int count,
                                          float (&acc)[kSweeps][kWide]) {
  constexpr int kTokens = kInFlight / kSweeps;
  for (int e0 = 0; e0 < count; e0 += kTokens) {
    typename Wide<TD>::Raw raw[kTokens][kSweeps];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      if (e0 + u < count) {
        const TD* row = dy + (int64_t)__builtin_amdgcn_readlane(token, e0 + u) * width;
#pragma unroll
        for (int s = 0; s < kSweeps; ++s)
          if (word + s * kLanes < words) raw[u][s] = Wide<TD>::load(row + (word + s * kLanes) * kWide);
      }
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      if (e0 + u < count) {
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) {
          if (word + s * kLanes < words) {
#pragma unroll
            for (int j = 0; j < kWide; ++j) acc[s][j] += Wide<TD>::get(raw[u][s], j);
          }
        }
      }
    }
  }
}

template <typename TD>
__device__ __forceinline__ float add_singles(const TD* dy, int64_t width, int64_t col, int token, int count) {
  float acc = 0.f;
  for (int e0 = 0; e0 < count; e0 += kInFlight) {
    float one[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (e0 + u < count) {
        const int64_t t = __builtin_amdgcn_readlane(token, e0 + u);
        if (col < width) one[u] = Wide<TD>::one(dy + t * width + col);
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (e0 + u < count && col < width) acc += one[u];
  }
  return acc;
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

// Sixteen bytes per lane and store, side by side.
template <typename TO>
__device__ __forceinline__ void zero_row(TO* at, int64_t width) {
  typedef typename Wide<TO>::Sixteen Sixteen;
  constexpr int kEach = 16 / (int)sizeof(TO);
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t pieces = width / kEach;
  RAFHIP_GLOBAL Sixteen* out = (RAFHIP_GLOBAL Sixteen*)at;
  for (int64_t w = lane; w < pieces; w += kLanes) out[w] = Sixteen{};
  const int64_t col = pieces * kEach + lane;
  if (col < width) Wide<TO>::put(at + col, 0.f);
}

// Calls f(sweeps, first word) until the wavefront has covered `words` words, two words per lane at a
// time where the row has them.
template <typename F>
__device__ __forceinline__ void for_words(int64_t words, F&& f) {
  int64_t w = 0;
  for (; words - w > kLanes; w += 2 * kLanes) f(std::integral_constant<int, 2>{}, w);
  if (words > w) f(std::integral_constant<int, 1>{}, w);
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
    // The set bits in ascending order: lane e learns the position of the e-th.
    int token[kRounds], count[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const uint64_t m = hits[k];
      const bool set = m >> lane & 1;
      const int place = __popcll(m & ((1ull << lane) - 1));
      count[k] = __popcll(m);
      // A lane that holds a token sends it to the lane of its rank, the others behind the last.
      token[k] = __builtin_amdgcn_ds_permute((set ? place : count[k] + (lane - place)) * 4, k * kLanes + lane);
    }
    const int64_t words = width / kWide;
    for_words(words, [&](auto sweeps, int64_t w) {
      constexpr int kSweeps = decltype(sweeps)::value;
      float acc[kSweeps][kWide] = {};
#pragma unroll
      for (int k = 0; k < kRounds; ++k) add_words<TD, kSweeps>(dy, width, w + lane, words, token[k], count[k], acc);
#pragma unroll
      for (int s = 0; s < kSweeps; ++s) {
        const int64_t word = w + lane + s * kLanes;
        if (word < words) put_row<TO, kWide>(at + word * kWide, acc[s], scale, accumulate != 0);
      }
    });
    const int64_t col = words * kWide + lane;
    if (words * kWide < width) {
      float acc[1] = {};
#pragma unroll
      for (int k = 0; k < kRounds; ++k) acc[0] += add_singles(dy, width, col, token[k], count[k]);
      if (col < width) put_row<TO, 1>(at + col, acc, scale, accumulate != 0);
    }
  }
}

// A wavefront takes kSlots rows.  kLanes / kSlots lanes for each row share the tiles, kRounds tiles a
// lane.  Rows without tokens become zeros, long ones are listed, and the tokens of the others go
// to the wavefront's own stretch of `entries`, row by row, kDirect of them for each row at most.
// Its rows lie `stride` apart: neighbours in a vocabulary are often alike in frequency, and a
// wavefront with eight rows of many tokens would finish long after the rest.
template <typename TO, int kSlots, int kRounds>
__global__ __launch_bounds__(kBlock) void find_rows(const uint32_t* keys, const uint16_t* index, int tiles, int tile_bits,
                                                    int bucket_bits, int buckets, int64_t stride, int64_t rows,
                                                    int64_t width, int accumulate, TO* dx, Taken* taken, uint32_t* entries_out,
                                                    uint32_t* counts, Item* singles, Item* items, Run* runs) {
  constexpr int kSpread = kLanes / kSlots;
  __shared__ uint32_t places[kWaves][kLanes];
  const int lane = threadIdx.x & (kLanes - 1);
  const int in_block = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + in_block;
  const int64_t n_waves = (int64_t)gridDim.x * kWaves;
  const uint32_t size = 1u << tile_bits;
  const int slot = lane / kSpread, tile0 = lane % kSpread;
  for (int64_t r0 = wave; r0 < stride; r0 += n_waves) {
    const int64_t my_row = r0 + slot * stride;
    uint32_t at[kRounds];
    int len[kRounds], before[kRounds];
    int total = 0;  // tokens of this lane's row, the same in all its lanes
    // Both ends of the row's run in each tile, by binary search in its bucket; the searches of a lane
    // go on side by side.
    uint32_t lo[kRounds], lo_end[kRounds], hi[kRounds], hi_end[kRounds];
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      const int t = q * kSpread + tile0;
      lo[q] = lo_end[q] = 0;
      if (my_row < rows && t < tiles) {
        const uint16_t* bucket = index + (int64_t)t * (buckets + 1) + (my_row >> bucket_bits);
        lo[q] = bucket[0];
        lo_end[q] = bucket[1];
      }
      hi[q] = lo[q];
      hi_end[q] = lo_end[q];
    }
    const uint32_t lo_key = (uint32_t)my_row << tile_bits, hi_key = (uint32_t)(my_row + 1) << tile_bits;
    for (bool more = true; more;) {
      more = false;
#pragma unroll
      for (int q = 0; q < kRounds; ++q) {
        const uint32_t* tile = keys + ((int64_t)(q * kSpread + tile0) << tile_bits);
        const uint32_t a = (lo[q] + lo_end[q]) >> 1, b = (hi[q] + hi_end[q]) >> 1;
        const uint32_t x = lo[q] < lo_end[q] ? tile[a] : 0, y = hi[q] < hi_end[q] ? tile[b] : 0;
        if (lo[q] < lo_end[q]) {
          if (x < lo_key)
            lo[q] = a + 1;
          else
            lo_end[q] = a;
        }
        if (hi[q] < hi_end[q]) {
          if (y < hi_key)
            hi[q] = b + 1;
          else
            hi_end[q] = b;
        }
        more |= lo[q] < lo_end[q] || hi[q] < hi_end[q];
      }
    }
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      at[q] = ((uint32_t)(q * kSpread + tile0) << tile_bits) + lo[q];
      len[q] = (int)(hi[q] - lo[q]);
    }
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      int sum = len[q];  // inclusive over the row's lanes
#pragma unroll
      for (int d = 1; d < kSpread; d <<= 1) {
        const int up = __shfl_up(sum, d, kSpread);
        if (tile0 >= d) sum += up;
      }
      before[q] = total + sum - len[q];
      total += __shfl(sum, kSpread - 1, kSpread);
    }
    int entries = 0, base = 0;  // tokens of the short rows; of those in front of this lane's row
    Taken want = 0;             // by the long ones
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int64_t row = r0 + i * stride;
      if (row >= rows) break;
      const int count = __builtin_amdgcn_readlane(total, i * kSpread);
      if (count <= kDirect) {
        if (count == 0 && !accumulate) zero_row(dx + row * width, width);
        if (slot == i) base = entries;
        entries += count;
        continue;
      }
      int n_runs = 0;
#pragma unroll
      for (int q = 0; q < kRounds; ++q) n_runs += __popcll(__ballot(slot == i && len[q] > 0));
      const int chunks = (count + kChunk - 1) / kChunk;
      want += take(n_runs, chunks);
    }
    if (want != 0) {
      Taken first = 0;
      if (lane == 0) first = atomicAdd(taken, want);
      first = (Taken)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)first) |
              (Taken)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(first >> 32)) << 32;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const int64_t row = r0 + i * stride;
        if (row >= rows) break;
        const int count = __builtin_amdgcn_readlane(total, i * kSpread);
        if (count <= kDirect) continue;
        const uint32_t first_run = runs_of(first);
        int n_runs = 0;
#pragma unroll
        for (int q = 0; q < kRounds; ++q) {
          const uint64_t some = __ballot(slot == i && len[q] > 0);
          if (slot == i && len[q] > 0)
            runs[first_run + n_runs + __popcll(some & ((1ull << lane) - 1))] = Run{at[q], (uint32_t)before[q]};
          n_runs += __popcll(some);
        }
        const int chunks = (count + kChunk - 1) / kChunk;
        Item* list = chunks == 1 ? singles + singles_of(first) : items + parts_of(first);
        for (int c = lane; c < chunks; c += kLanes)
          list[c] = Item{(uint32_t)row, (uint32_t)count, (uint32_t)n_runs, first_run, (uint32_t)c};
        first += take(n_runs, chunks);
      }
    }
    if (lane == 0) counts[r0] = (uint32_t)entries;
    if (entries == 0) continue;
    // Lane e gets the e-th token of the short rows.
    if (total <= kDirect) {
#pragma unroll
      for (int q = 0; q < kRounds; ++q)
        for (int x = 0; x < len[q]; ++x) places[in_block][base + before[q] + x] = (at[q] + x) | (uint32_t)slot << kSlotShift;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (lane < entries) {
      const uint32_t place = places[in_block][lane], key_at = place & ((1u << kSlotShift) - 1);
      const uint32_t token = (key_at >> tile_bits << tile_bits) + (keys[key_at] & (size - 1));
      entries_out[r0 * (kSlots * kDirect) + lane] = token | (place >> kSlotShift << kSlotShift);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// The short rows of one wavefront of find_rows: `entries` tokens, one per lane, in one go, so that the
// loads of the next row are under way while this one is finished.
template <typename TD, typename TO>
__device__ __forceinline__ void sum_short_rows(const TD* dy, int64_t width, uint32_t entry, int entries, int64_t r0,
                                               int64_t stride, float scale, bool accumulate, TO* dx) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t words = width / kWide;
  const int token = (int)(entry & ((1u << kSlotShift) - 1)), of = (int)(entry >> kSlotShift);
  const int next = __shfl_down(of, 1, kLanes);
  const uint64_t last = __ballot(lane < entries && (lane + 1 == entries || next != of));  // of its row
  for_words(words, [&](auto sweeps, int64_t w) {
    constexpr int kSweeps = decltype(sweeps)::value;
    constexpr int kTokens = kInFlight / kSweeps;
    const int64_t word = w + lane;
    float acc[kSweeps][kWide] = {};
    for (int e0 = 0; e0 < entries; e0 += kTokens) {
      typename Wide<TD>::Raw raw[kTokens][kSweeps];
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        if (e0 + u < entries) {
          const TD* row = dy + (int64_t)__builtin_amdgcn_readlane(token, e0 + u) * width;
#pragma unroll
          for (int s = 0; s < kSweeps; ++s)
            if (word + s * kLanes < words) raw[u][s] = Wide<TD>::load(row + (word + s * kLanes) * kWide);
        }
      }
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        if (e0 + u < entries) {
          const bool done = last >> (e0 + u) & 1;
          TO* out = dx + (r0 + __builtin_amdgcn_readlane(of, e0 + u) * stride) * width;
#pragma unroll
          for (int s = 0; s < kSweeps; ++s) {
            if (word + s * kLanes < words) {
#pragma unroll
              for (int j = 0; j < kWide; ++j) acc[s][j] += Wide<TD>::get(raw[u][s], j);
              if (done) {
                put_row<TO, kWide>(out + (word + s * kLanes) * kWide, acc[s], scale, accumulate);
#pragma unroll
                for (int j = 0; j < kWide; ++j) acc[s][j] = 0.f;
              }
            }
          }
        }
      }
    }
  });
  const int64_t col = words * kWide + lane;  // columns behind the last whole word
  if (words * kWide < width) {
    float acc[1] = {0.f};
    for (int e = 0; e < entries; ++e) {
      const int64_t t = __builtin_amdgcn_readlane(token, e);
      const int64_t row = r0 + __builtin_amdgcn_readlane(of, e) * stride;
      if (col < width) {
        acc[0] += Wide<TD>::one(dy + t * width + col);
        if (last >> e & 1) {
          put_row<TO, 1>(dx + row * width + col, acc, scale, accumulate);
          acc[0] = 0.f;
        }
      }
    }
  }
}

// The first chunk_blocks workgroups take the chunks, one after the other: each of eight wavefronts sums
// kPerWave tokens, the sums are added in order, and the result is the row (a row of one chunk) or a
// partial sum.  The others take the short rows.
template <typename TD, typename TO>
__global__ __launch_bounds__(kChunkBlock) void sum_rows(const TD* dy, const uint32_t* keys, int tile_bits, int64_t width,
                                                        float scale, int accumulate, TO* dx, const Taken* taken,
                                                        const uint32_t* entries, const uint32_t* counts, int64_t stride,
                                                        int per_wave, const Item* singles, const Item* items,
                                                        const Run* runs, float* parts, unsigned chunk_blocks) {
  constexpr int kSweeps = 1;
  __shared__ float sums[kChunkWaves][kLanes * kWide];
  const int lane = threadIdx.x & (kLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  if (blockIdx.x >= chunk_blocks) {
    const int64_t n_waves = (int64_t)(gridDim.x - chunk_blocks) * kChunkWaves;
    for (int64_t r0 = (int64_t)(blockIdx.x - chunk_blocks) * kChunkWaves + wave; r0 < stride; r0 += n_waves) {
      const int count = __builtin_amdgcn_readfirstlane((int)counts[r0]);
      const uint32_t entry = lane < per_wave ? entries[r0 * per_wave + lane] : 0;  // what lies behind the last is not used
      if (count > 0) sum_short_rows(dy, width, entry, count, r0, stride, scale, accumulate != 0, dx);
    }
    return;
  }
  const Taken listed = *taken;
  const uint32_t n_parts = parts_of(listed), n_items = n_parts + singles_of(listed);
  const int64_t words = width / kWide;
  for (uint32_t it = blockIdx.x; it < n_items; it += chunk_blocks) {
    const Item item = it < n_parts ? items[it] : singles[it - n_parts];
    const int first = (int)item.chunk * kChunk + wave * kPerWave;
    int count = (int)item.tokens - first;
    count = count < 0 ? 0 : count > kPerWave ? kPerWave : count;
    // Where this lane's token is: in the last run that starts at or before it.
    const uint32_t want = (uint32_t)(first + lane);
    uint32_t at = 0, before = 0;
    for (uint32_t r0 = 0; r0 < item.n_runs && count > 0; r0 += kLanes) {
      Run mine{0, 0xffffffffu};
      if (r0 + lane < item.n_runs) mine = runs[item.first_run + r0 + lane];
#pragma unroll
      for (int e = 0; e < kPerWave; ++e) {
        const uint64_t started = __ballot(mine.before <= (uint32_t)(first + e));
        if (started != 0) {
          const int last = 63 - __clzll((long long)started);
          const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)mine.at, last);
          const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)mine.before, last);
          if (lane == e) {
            at = a;
            before = b;
          }
        }
      }
    }
    int token = 0;
    if (lane < count) {
      const uint32_t key_at = at + (want - before);
      token = (int)((key_at >> tile_bits << tile_bits) + (keys[key_at] & ((1u << tile_bits) - 1)));
    }
    const bool whole = it >= n_parts;
    float* part = parts + (int64_t)it * width;
    TO* out = dx + (int64_t)item.row * width;
    // `n` columns from `col` on, each the sum of the wavefronts' in order.
    auto join = [&](int64_t col, int n) {
      __syncthreads();
      for (int c = threadIdx.x; c < n; c += kChunkBlock) {
        float total[1] = {sums[0][c]};
#pragma unroll
        for (int k = 1; k < kChunkWaves; ++k) total[0] += sums[k][c];
        if (whole)
          put_row<TO, 1>(out + col + c, total, scale, accumulate != 0);
        else
          part[col + c] = total[0];
      }
      __syncthreads();
    };
    for (int64_t w = 0; w < words; w += kLanes) {
      float acc[kSweeps][kWide] = {};
      add_words<TD, kSweeps>(dy, width, w + lane, words, token, count, acc);
#pragma unroll
      for (int j = 0; j < kWide; ++j) sums[wave][lane * kWide + j] = acc[0][j];
      const int64_t left = (words - w) * kWide;
      join(w * kWide, (int)(left < kLanes * kWide ? left : kLanes * kWide));
    }
    if (words * kWide < width) {
      sums[wave][lane] = add_singles(dy, width, words * kWide + lane, token, count);
      join(words * kWide, (int)(width - words * kWide));
    }
  }
}

// The chunks of a long row added in order: 64 columns per workgroup, four stretches of chunks.
template <typename TO>
__global__ __launch_bounds__(kBlock) void join_chunks(int64_t width, float scale, int accumulate, TO* dx,
                                                     const Taken* taken, const Item* items, const float* parts) {
  __shared__ float sums[kWaves][kLanes];
  const int lane = threadIdx.x & (kLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t col = (int64_t)blockIdx.x * kLanes + lane;
  const uint32_t n_parts = parts_of(*taken);
  for (uint32_t it = blockIdx.y; it < n_parts; it += gridDim.y) {
    const Item row = items[it];
    if (row.chunk != 0) continue;  // the first chunk stands for its row
    const int chunks = (int)((row.tokens + kChunk - 1) / kChunk);
    const int per = (chunks + kWaves - 1) / kWaves;
    const int from = wave * per, to = from + per < chunks ? from + per : chunks;
    float acc = 0.f;
    if (col < width) {
      const float* p = parts + (int64_t)it * width + col;
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
constexpr int64_t kMaxFindBlocks = 2048;  // eight per CU; a launch of more would only take longer to start
constexpr int64_t kMaxSumBlocks = 1024;   // four of twice the size

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
  auto* taken = reinterpret_cast<Taken*>(ws + l.taken_at);
  auto* keys = reinterpret_cast<uint32_t*>(ws + l.keys_at);
  auto* index = reinterpret_cast<uint16_t*>(ws + l.index_at);
  auto* entries = reinterpret_cast<uint32_t*>(ws + l.entries_at);
  auto* counts = reinterpret_cast<uint32_t*>(ws + l.counts_at);
  auto* singles = reinterpret_cast<Item*>(ws + l.singles_at);
  auto* items = reinterpret_cast<Item*>(ws + l.items_at);
  auto* runs = reinterpret_cast<Run*>(ws + l.runs_at);
  auto* parts = reinterpret_cast<float*>(ws + l.parts_at);
  auto sort = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)l.tiles), dim3(kSortBlock), 0, s, ids, n, which, l.tile_bits, l.bucket_bits,
                       l.buckets, keys, index, taken);
  };
  switch (l.tile_bits) {
    case 11: sort(tile_sort<Id, 2>); break;
    case 12: sort(tile_sort<Id, 4>); break;
    case 13: sort(tile_sort<Id, 8>); break;
    default: sort(tile_sort<Id, 16>); break;
  }
  const int group = l.tiles <= kLanes ? kGroup : 1;
  const int64_t waves = (rows + group - 1) / group;  // of find_rows, and the distance of a wavefront's rows
  const int64_t max_blocks = (waves + kWaves - 1) / kWaves;
  const unsigned find_blocks = (unsigned)(max_blocks < kMaxFindBlocks ? max_blocks : kMaxFindBlocks);
  auto find = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(find_blocks), dim3(kBlock), 0, s, keys, index, l.tiles, l.tile_bits, l.bucket_bits,
                       l.buckets, waves, rows, width, accumulate, dx, taken, entries, counts, singles, items, runs);
  };
  if (l.tiles <= 8)
    find(find_rows<TO, kGroup, 1>);
  else if (l.tiles <= 32)
    find(find_rows<TO, kGroup, 4>);
  else if (l.tiles <= kLanes)
    find(find_rows<TO, kGroup, 8>);
  else
    find(find_rows<TO, 1, kMaxTiles / kLanes>);
  const int64_t max_items = l.max_singles + l.max_parts, max_short = (waves + kChunkWaves - 1) / kChunkWaves;
  const unsigned chunk_blocks = (unsigned)(max_items < kMaxSumBlocks ? max_items : kMaxSumBlocks);
  const unsigned short_blocks = (unsigned)(max_short < kMaxSumBlocks ? max_short : kMaxSumBlocks);
  hipLaunchKernelGGL((sum_rows<TD, TO>), dim3(chunk_blocks + short_blocks), dim3(kChunkBlock), 0, s, dy, keys, l.tile_bits,
                     width, scale, accumulate, dx, taken, entries, counts, waves, group * kDirect, singles, items, runs,
                     parts, chunk_blocks);
  hipLaunchKernelGGL(join_chunks<TO>, dim3((unsigned)((width + kLanes - 1) / kLanes), (unsigned)(l.max_parts < 256 ? l.max_parts : 256)),
                     dim3(kBlock), 0, s, width, scale, accumulate, dx, taken, items, parts);
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
