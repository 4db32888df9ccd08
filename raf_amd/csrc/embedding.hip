// Token embedding and its gradient for gfx950: `raf.op.embedding` / `raf.op.embedding_dx`
// (src/op/dialect/cuda/embedding.cc in the reference, which gathers and scatters unscaled rows).
//
// Forward: y[t] = scale * x[ids[t]], a gather that reads and writes each element once.
//
// Gradient: dx[r] = scale * sum over the tokens of row r of dy[t].  A sum by floating-point atomics
// would depend on the order in which they arrive, so tokens are sorted by row first:
//   1. tile_sort   sorts each tile of tokens by (row, position)
//                  (meanwhile the gradient is zeroed, if most rows will have no tokens);
//   2. find_rows   looks every row up in all sorted tiles at once (a binary search per lane and
//                  tile), else writes zeros for rows without tokens, and lists the others: the tokens of
//                  rows of up to kDirect, and chunks of kChunk tokens of longer rows;
//   3. sum_rows    sums what is listed, a wavefront for 64 words of a chunk or of eight short rows, so
//                  that a token that fills half the batch is spread over the GPU;
//   4. join_chunks adds the chunks of a row in order.
// Runs of a row are visited in tile order and sorted inside a tile, so every sum runs over
// ascending positions cut at multiples of kChunk: the result depends on the data alone although
// the list of long rows is filled in the order in which wavefronts arrive.  Up to kFewTokens
// tokens one launch does it all, every wavefront looking through all the ids.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_table.h"
#include "rafhip_vocab.h"
#include "status.h"
#include "vocab_io.h"

namespace rafhip {
namespace {

constexpr int kBlock = 256;
constexpr int kLanes = 64;
constexpr int kWaves = kBlock / kLanes;

// ------------------------------------------------------------------------------------- forward
// The product as an fp32 number.  For fp16 the compiler would else pick an instruction that rounds the
// product to 16 bits at once, and only there: the other types' values are rounded to fp32 first.
__device__ __forceinline__ float scaled(float scale, float x) {
  float y = scale * x;
  asm volatile("" : "+v"(y));
  return y;
}

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
    bool inside[kInFlight];
    // Loads without a condition: a place behind the last repeats it, and for an index outside the
    // table the word comes from row 0, which exists here, and is not used.  (The compiler puts a
    // wait for all earlier loads in front of every load in a branch.)
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const unsigned i = i0 + u * kBlock < items ? i0 + u * kBlock : items - 1;
      const unsigned t = i / (unsigned)words, c = i - t * (unsigned)words;
      const uint64_t row = (uint64_t)(int64_t)ids[t0 + t] - (uint64_t)first_row;
      inside[u] = row < (uint64_t)rows;
      to[u] = (t0 + t) * width + (int64_t)c * kWide;
      raw[u] = Wide<TX>::load(x + (inside[u] ? (int64_t)row : 0) * width + (int64_t)c * kWide);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (i0 + u * kBlock < items) {
        float v[kWide];
#pragma unroll
        for (int j = 0; j < kWide; ++j) v[j] = inside[u] ? scaled(scale, Wide<TX>::get(raw[u], j)) : 0.f;
        Wide<TY>::store(y + to[u], v);
      }
    }
  }
  const int rest = (int)(width - (int64_t)words * kWide);  // columns behind the last whole word
  const unsigned singles = (unsigned)tokens * (unsigned)rest;
  for (unsigned i = threadIdx.x; i < singles; i += kBlock) {
    const unsigned t = i / (unsigned)rest, c = i - t * (unsigned)rest;
    const uint64_t row = (uint64_t)(int64_t)ids[t0 + t] - (uint64_t)first_row;
    const int64_t col = (int64_t)words * kWide + c;
    const float v = row < (uint64_t)rows ? scaled(scale, Wide<TX>::one(x + (int64_t)row * width + col)) : 0.f;
    Wide<TY>::put(y + (t0 + t) * width + col, v);
  }
}

// The rows of an empty table: zeros.
template <typename TY>
__global__ __launch_bounds__(kBlock) void no_rows(TY* y, int64_t elements) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < elements; i += (int64_t)gridDim.x * kBlock)
    Wide<TY>::put(y + i, 0.f);
}

// ------------------------------------------------------------------------------------ gradient
constexpr int kFewTokens = 256;  // one launch up to here
constexpr int kDirect = 8;       // tokens of a row that one wavefront sums
constexpr int kChunk = 32;       // tokens of one partial sum of a longer row
constexpr int kMinTileBits = 10, kMaxTileBits = 14;
constexpr int kMaxTiles = 512;
constexpr int kGroup = kLanes / kDirect;  // rows of a wavefront: their tokens have a lane each
constexpr int kSmallSort = 512, kSort = 1024;  // threads of a tile of 2^10 tokens, of more
constexpr int kInFlight = 8;  // words in flight per lane
// Of a chunk: a short batch waits for its round trips (3003 tokens 31.3 us with two of 16, 33.3 with four of 8).
constexpr int kChunkInFlight = 16;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr int kSlotShift = 28;  // an entry: a token (23 bits: kMaxTiles tiles of 2^14) and its row's slot

struct Layout {
  int tile_bits = 0;
  int tiles = 0;
  int bucket_bits = 0;  // log2 of the rows that share an entry of a tile's index
  int buckets = 0;
  int64_t max_singles = 0;  // rows of more than kDirect tokens and no more than a chunk
  int64_t max_runs = 0;   // runs of them
  int64_t max_long = 0;   // rows of more than one chunk
  int64_t max_parts = 0;  // their chunks
  int64_t keys_at = 0, index_at = 0, taken_at = 0, entries_at = 0, counts_at = 0, singles_at = 0, items_at = 0;
  int64_t long_at = 0, runs_at = 0, parts_at = 0, bytes = 0;
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
// (with four, 800 wavefronts queued for 60 us).
typedef unsigned long long Taken;
constexpr int kRunBits = 24, kSingleBits = 21;  // up to 2^23 runs, 2^23 / 9 rows of one chunk, 2^23 / 16 chunks
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
  l->max_long = n / (kChunk + 1);
  l->max_parts = n / kChunk + l->max_long;
  auto place = [&](int64_t bytes) {
    const int64_t at = l->bytes;
    l->bytes += align256(bytes);
    return at;
  };
  l->taken_at = place(2 * sizeof(Taken));  // and how many rows of more than one chunk there are
  l->keys_at = place((tiles << bits) * 4);
  // About one key per entry, or 16 rows where the keys are many: a search then takes a step or two.
  int bucket = row_bits - bits;
  if (bucket < 4) bucket = 4;
  l->bucket_bits = bucket;
  l->buckets = (int)((rows + (1LL << bucket) - 1) >> bucket);
  l->index_at = place(tiles * (l->buckets + 1) * 2);
  l->entries_at = place(rows * kDirect * 4);
  l->counts_at = place(rows * 4);
  l->singles_at = place(l->max_singles * (int64_t)sizeof(Item));
  l->items_at = place(l->max_parts * (int64_t)sizeof(Item));
  l->long_at = place(l->max_long * 4);
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

// The value of the lane whose number differs in the bit kMask: without LDS where the lanes are within
// 16 of each other.
template <int kMask>
__device__ __forceinline__ uint32_t from_lane_xor(uint32_t x) {
  if constexpr (kMask == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);   // quad_perm 1 0 3 2
  if constexpr (kMask == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  if constexpr (kMask == 4) {  // 7 - i of each eight, then 3 - i of each four
    const int y = __builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true);
    return (uint32_t)__builtin_amdgcn_mov_dpp(y, 0x1b, 0xf, 0xf, true);
  }
  if constexpr (kMask == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true);  // row_ror 8 of 16
  return (uint32_t)__shfl_xor((int)x, kMask, kLanes);
}

template <int kEach, int kMask>
__device__ __forceinline__ void exchange_lanes(uint32_t (&v)[kEach], int tid, int k) {
  if (kMask * kEach >= k) return;
  const bool low = (tid & kMask) == 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t y = from_lane_xor<kMask>(v[e]);
    const bool up = ((tid * kEach + e) & k) == 0;
    v[e] = low == up ? min(v[e], y) : max(v[e], y);
  }
}

// Zeros to `bytes` bytes, of which a multiple of 16 of a 2-byte aligned address, by `block` of `blocks` workgroups.
__device__ __forceinline__ void fill_zeros(char* at, int64_t bytes, int64_t block, int64_t blocks) {
  typedef uint32_t Sixteen __attribute__((ext_vector_type(4)));
  int64_t head = (int64_t)(-(intptr_t)at & 15);
  head = head < bytes ? head : bytes;
  const int64_t pieces = (bytes - head) / 16, done = head + pieces * 16;
  RAFHIP_GLOBAL Sixteen* out = (RAFHIP_GLOBAL Sixteen*)(at + head);
  for (int64_t i = block * blockDim.x + threadIdx.x; i < pieces; i += blocks * blockDim.x) out[i] = Sixteen{};
  const int64_t i = 2 * (int64_t)threadIdx.x;  // the ends, fewer than 16 bytes each
  if (block == 0 && i < head) *(RAFHIP_GLOBAL uint16_t*)(at + i) = 0;
  if (block == 0 && i < bytes - done) *(RAFHIP_GLOBAL uint16_t*)(at + done + i) = 0;
}

// Sorts one tile by a bitonic network over (row << tile_bits | position), kEach keys in the registers
// of each thread: key i sits in register i % kEach of thread i / kEach, so of the 55 stages of 1024
// keys 10 stay inside a thread, 39 inside a wavefront and 6 go through LDS.  Then the index: for every
// bucket of rows the first key that is not below it.  Workgroups behind the tiles write fill_bytes of zeros.
template <typename Id, int kThreads, int kEach>
__global__ __launch_bounds__(kThreads) void tile_sort(const Id* ids, int64_t n, Which which, int tile_bits,
                                                      int bucket_bits, int buckets, uint32_t* keys, uint16_t* index,
                                                      Taken* taken, int tiles, char* fill, int64_t fill_bytes) {
  if ((int)blockIdx.x >= tiles) return fill_zeros(fill, fill_bytes, (int)blockIdx.x - tiles, (int)gridDim.x - tiles);
  constexpr int kSize = kEach * kThreads;
  __shared__ uint32_t lds[kSize];
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * kSize;
  if (blockIdx.x == 0 && tid < 2) taken[tid] = 0;
  uint32_t v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kThreads + tid;  // any order will do before the sort
    const int64_t row = t0 + i < n ? which.row((int64_t)ids[t0 + i]) : -1;
    v[e] = row >= 0 ? (uint32_t)row << tile_bits | (uint32_t)i : kNoToken;
  }
#pragma unroll 1
  for (int k = 2; k <= kSize; k <<= 1) {
    for (int j = k >> 1; j >= kEach * kLanes; j >>= 1) {  // across wavefronts
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) lds[e * kThreads + tid] = v[e];
      __syncthreads();
      const int other = tid ^ (j / kEach);
      const bool low = (tid & (j / kEach)) == 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const uint32_t y = lds[e * kThreads + other];
        const bool up = ((tid * kEach + e) & k) == 0;
        v[e] = low == up ? min(v[e], y) : max(v[e], y);
      }
    }
    exchange_lanes<kEach, 32>(v, tid, k);
    exchange_lanes<kEach, 16>(v, tid, k);
    exchange_lanes<kEach, 8>(v, tid, k);
    exchange_lanes<kEach, 4>(v, tid, k);
    exchange_lanes<kEach, 2>(v, tid, k);
    exchange_lanes<kEach, 1>(v, tid, k);
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
  for (int i = tid; i < kSize; i += kThreads) keys[t0 + i] = lds[i];
  for (int b = tid; b <= buckets; b += kThreads) {
    // The last entry lies behind every row; its key may exceed 32 bits.
    const uint64_t key = (uint64_t)b << (bucket_bits + tile_bits);
    int at = 0;
    for (int step = kSize >> 1; step > 0; step >>= 1)
      if (lds[at + step - 1] < key) at += step;
    at += lds[at] < key ? 1 : 0;
    index[(int64_t)blockIdx.x * (buckets + 1) + b] = (uint16_t)at;
  }
}

// Words kSweeps times 64 apart of `count` > 0 tokens, of which lane e of `token` holds the e-th, added to
// acc; `count` is the same in all lanes.  The loads are issued without a condition -- lanes behind
// the row's last word and places behind the last token repeat that one -- because the compiler puts
// a wait for all earlier loads in front of every load in a branch.
template <typename TD, int kSweeps, int kTokens>
__device__ __forceinline__ void add_words(const TD* dy, int64_t width, int64_t word, int64_t words, int token, int count,
                                          float (&acc)[kSweeps][kWide]) {
  for (int e0 = 0; e0 < count; e0 += kTokens) {
    typename Wide<TD>::Raw raw[kTokens][kSweeps];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int e = e0 + u < count ? e0 + u : count - 1;
      const TD* row = dy + (int64_t)__builtin_amdgcn_readlane(token, e) * width;
#pragma unroll
      for (int s = 0; s < kSweeps; ++s) {
        const int64_t w = word + s * kLanes;
        raw[u][s] = Wide<TD>::load(row + (w < words ? w : words - 1) * kWide);
      }
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      if (e0 + u < count) {
#pragma unroll
        for (int s = 0; s < kSweeps; ++s) {
#pragma unroll
          for (int j = 0; j < kWide; ++j) acc[s][j] += Wide<TD>::get(raw[u][s], j);
        }
      }
    }
  }
}

template <typename TD>
__device__ __forceinline__ float add_singles(const TD* dy, int64_t width, int64_t col, int token, int count) {
  float acc = 0.f;
  if (col >= width) col = width - 1;
  for (int e0 = 0; e0 < count; e0 += kInFlight) {
    float one[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int64_t t = __builtin_amdgcn_readlane(token, e0 + u < count ? e0 + u : count - 1);
      one[u] = Wide<TD>::one(dy + t * width + col);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (e0 + u < count) acc += one[u];
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

// The tokens of a row among up to kFewTokens, as bits, summed into the row by a wavefront.
template <typename TD, typename TO, int kRounds>
__device__ __forceinline__ void sum_hits(const TD* dy, int64_t width, const uint64_t (&hits)[kRounds], float scale,
                                         bool accumulate, TO* at) {
  const int lane = threadIdx.x & (kLanes - 1);
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
    for (int k = 0; k < kRounds; ++k)
      add_words<TD, kSweeps, kInFlight / kSweeps>(dy, width, w + lane, words, token[k], count[k], acc);
#pragma unroll
    for (int s = 0; s < kSweeps; ++s) {
      const int64_t word = w + lane + s * kLanes;
      if (word < words) put_row<TO, kWide>(at + word * kWide, acc[s], scale, accumulate);
    }
  });
  const int64_t col = words * kWide + lane;
  if (words * kWide < width) {
    float acc[1] = {};
#pragma unroll
    for (int k = 0; k < kRounds; ++k) acc[0] += add_singles(dy, width, col, token[k], count[k]);
    if (col < width) put_row<TO, 1>(at + col, acc, scale, accumulate);
  }
}

// All of the gradient for up to kFewTokens tokens.  Written anew, a wavefront takes rows_per_wave rows and looks
// through all the ids for them; added to (rows_per_wave 0), it takes a token and sums those of its
// row if it is the first of them (37 tokens, 30522 x 768 rows: 8.8 us by rows, 4.4 by tokens).
template <typename TD, typename TO, typename Id>
__global__ __launch_bounds__(kBlock) void few_tokens(const TD* dy, const Id* ids, int n, Which which, int64_t width,
                                                     float scale, int rows_per_wave, TO* dx) {
  constexpr int kRounds = kFewTokens / kLanes;
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const bool accumulate = rows_per_wave == 0;
  const int64_t r0 = wave * rows_per_wave;
  if (accumulate ? wave >= n : r0 >= which.rows) return;
  const int mine = (int)(which.rows - r0 < rows_per_wave ? which.rows - r0 : rows_per_wave);
  int64_t row[kRounds];
  bool any = false;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int t = k * kLanes + lane;
    const int64_t r = n > 0 ? which.row((int64_t)ids[t < n ? t : n - 1]) : -1;
    row[k] = t < n && r >= 0 ? r - r0 : -1;
    any |= row[k] >= 0 && row[k] < mine;
  }
  if (accumulate) {
    const int64_t r = which.row((int64_t)ids[wave]);
    if (r < 0) return;
    uint64_t hits[kRounds], earlier = 0;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      hits[k] = __ballot(row[k] == r);
      const int64_t before = wave - k * kLanes;  // of these tokens, those in front of this wavefront's
      earlier |= before <= 0 ? 0 : before >= kLanes ? hits[k] : hits[k] & ((1ull << before) - 1);
    }
    if (earlier == 0) sum_hits<TD, TO, kRounds>(dy, width, hits, scale, true, dx + r * width);
    return;
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
    if (all == 0)
      zero_row(at, width);
    else
      sum_hits<TD, TO, kRounds>(dy, width, hits, scale, false, at);
  }
}

// Element i of a list whose bytes 32 bits can count: the address is one register behind a base.
template <typename T>
__device__ __forceinline__ T element(const T* base, uint32_t i) {
  return *(const RAFHIP_GLOBAL T*)((const char*)base + (size_t)(i * (uint32_t)sizeof(T)));
}

// A wavefront takes kSlots neighbouring rows, whose places in a tile are neighbours too.  kLanes /
// kSlots lanes for each row share the tiles, kRounds tiles a lane.  Rows without tokens become
// zeros, long ones are listed, and the tokens of the others go to entries[row][kDirect].
template <typename TO, int kSlots, int kRounds>
__global__ __launch_bounds__(kBlock) void find_rows(const uint32_t* keys, const uint16_t* index, int tiles, int tile_bits,
                                                    int bucket_bits, int buckets, int64_t rows, int64_t width,
                                                    int write_zeros, TO* dx, Taken* taken, uint32_t* entries,
                                                    uint32_t* counts, Item* singles, Item* items, uint32_t* long_rows,
                                                    Run* runs) {
  constexpr int kSpread = kLanes / kSlots;
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t n_waves = (int64_t)gridDim.x * kWaves;
  const uint32_t size = 1u << tile_bits;
  const int slot = lane / kSpread, tile0 = lane % kSpread;
  for (int64_t r0 = wave * kSlots; r0 < rows; r0 += n_waves * kSlots) {
    const int64_t my_row = r0 + slot;
    uint32_t at[kRounds];
    int len[kRounds], before[kRounds];
    int total = 0;  // tokens of this lane's row, the same in all its lanes
    // Both ends of the row's run in each tile, by binary search in its bucket; the searches of a lane
    // go on side by side.
    uint32_t lo[kRounds], lo_end[kRounds], hi[kRounds], hi_end[kRounds];
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      // Loads without a condition here and below: lanes without a tile or a row look at the first
      // tile or the last row.
      const int t = q * kSpread + tile0 < tiles ? q * kSpread + tile0 : 0;
      const uint16_t* bucket = index + (int64_t)t * (buckets + 1) + ((my_row < rows ? my_row : rows - 1) >> bucket_bits);
      lo[q] = bucket[0];
      lo_end[q] = bucket[1];
    }
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      if (my_row >= rows || q * kSpread + tile0 >= tiles) lo[q] = lo_end[q] = 0;
      hi[q] = lo[q];
      hi_end[q] = lo_end[q];
    }
    const uint32_t lo_key = (uint32_t)my_row << tile_bits, hi_key = (uint32_t)(my_row + 1) << tile_bits;
    for (bool more = true; more;) {
      more = false;
      uint32_t x[kRounds], y[kRounds];
#pragma unroll
      for (int q = 0; q < kRounds; ++q) {
        const uint32_t tile = (uint32_t)(q * kSpread + tile0 < tiles ? q * kSpread + tile0 : 0) << tile_bits;
        const uint32_t a = (lo[q] + lo_end[q]) >> 1, b = (hi[q] + hi_end[q]) >> 1;  // size where the run ends the tile
        x[q] = element(keys, tile + (a < size ? a : 0));
        y[q] = element(keys, tile + (b < size ? b : 0));
      }
#pragma unroll
      for (int q = 0; q < kRounds; ++q) {
        const uint32_t a = (lo[q] + lo_end[q]) >> 1, b = (hi[q] + hi_end[q]) >> 1;
        if (lo[q] < lo_end[q]) {
          if (x[q] < lo_key)
            lo[q] = a + 1;
          else
            lo_end[q] = a;
        }
        if (hi[q] < hi_end[q]) {
          if (y[q] < hi_key)
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
    if (my_row < rows && total <= kDirect) {
      if (tile0 == 0) counts[my_row] = (uint32_t)total;
      uint32_t key[kRounds];  // of the first token of each run; most runs have no other
#pragma unroll
      for (int q = 0; q < kRounds; ++q) key[q] = element(keys, len[q] > 0 ? at[q] : 0);
#pragma unroll
      for (int q = 0; q < kRounds; ++q) {
        const uint32_t first_of_tile = (uint32_t)(q * kSpread + tile0) << tile_bits;
        uint32_t* out = entries + my_row * kDirect + before[q];
        if (len[q] > 0) out[0] = first_of_tile + (key[q] & (size - 1));
        for (int x = 1; x < len[q]; ++x) out[x] = first_of_tile + (element(keys, at[q] + x) & (size - 1));
      }
    } else if (my_row < rows && tile0 == 0) {
      counts[my_row] = 0;
    }
    Taken want = 0;  // by the long rows
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int64_t row = r0 + i;
      if (row >= rows) break;
      const int count = __builtin_amdgcn_readlane(total, i * kSpread);
      if (count <= kDirect) {
        if (count == 0 && write_zeros) zero_row(dx + row * width, width);
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
        const int64_t row = r0 + i;
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
        if (chunks > 1 && lane == 0) long_rows[atomicAdd((uint32_t*)(taken + 1), 1u)] = parts_of(first);
        first += take(n_runs, chunks);
      }
    }
  }
}

// A slice of 64 words of kGroup rows, `stride` apart, by a wavefront: the tokens of the short ones, a lane for each, in one go,
// so that the loads of the next row are under way while this one is finished.  Neighbours in a
// vocabulary are often alike in frequency; a wavefront with eight neighbouring rows of many tokens
// would finish long after the rest.
template <typename TD, typename TO>
__device__ __forceinline__ void sum_short_rows(const TD* dy, int64_t width, const uint32_t* entry, const uint32_t* counts,
                                               int64_t r0, int64_t stride, int64_t rows, int slice, float scale,
                                               bool accumulate, TO* dx) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int slot = lane / kDirect, x = lane % kDirect;
  const int64_t my_row = r0 + slot * stride;
  const bool set = my_row < rows && x < (int)counts[my_row < rows ? my_row : 0];
  const uint32_t mine = set ? entry[my_row * kDirect + x] | (uint32_t)slot << kSlotShift : 0;
  const uint64_t m = __ballot(set);
  const int entries = __popcll(m);
  if (entries == 0) return;
  // A lane that holds a token sends it to the lane of its rank, the others behind the last.
  const int rank = __popcll(m & ((1ull << lane) - 1));
  const uint32_t got = (uint32_t)__builtin_amdgcn_ds_permute((set ? rank : entries + (lane - rank)) * 4, (int)mine);
  const int token = (int)(got & ((1u << kSlotShift) - 1)), of = (int)(got >> kSlotShift);
  const int64_t words = width / kWide;
  const int next = __shfl_down(of, 1, kLanes);
  const uint64_t last = __ballot(lane < entries && (lane + 1 == entries || next != of));  // of its row
  const int64_t word = (int64_t)slice * kLanes + lane;
  float acc[kWide] = {};
  // A batch of kTokens, loads first and without a condition, as in add_words.
  auto batch = [&](auto tokens, int e0) {
    constexpr int kTokens = decltype(tokens)::value;
    typename Wide<TD>::Raw raw[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int e = e0 + u < entries ? e0 + u : entries - 1;
      const TD* row = dy + (int64_t)__builtin_amdgcn_readlane(token, e) * width;
      raw[u] = Wide<TD>::load(row + (word < words ? word : words - 1) * kWide);
    }
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      if (e0 + u < entries) {
#pragma unroll
        for (int j = 0; j < kWide; ++j) acc[j] += Wide<TD>::get(raw[u], j);
        if (last >> (e0 + u) & 1) {
          TO* out = dx + (r0 + __builtin_amdgcn_readlane(of, e0 + u) * stride) * width;
          if (word < words) put_row<TO, kWide>(out + word * kWide, acc, scale, accumulate);
#pragma unroll
          for (int j = 0; j < kWide; ++j) acc[j] = 0.f;
        }
      }
    }
  };
  if ((int64_t)slice * kLanes < words) {
    int e0 = 0;
    for (; entries - e0 > kInFlight / 2; e0 += kInFlight) batch(std::integral_constant<int, kInFlight>{}, e0);
    if (e0 < entries) batch(std::integral_constant<int, kInFlight / 2>{}, e0);
  }
  const int64_t col = words * kWide + lane;  // columns behind the last whole word
  if (slice == 0 && words * kWide < width) {
    float one[1] = {0.f};
    for (int e = 0; e < entries; ++e) {
      const int64_t t = __builtin_amdgcn_readlane(token, e);
      const int64_t row = r0 + __builtin_amdgcn_readlane(of, e) * stride;
      if (col < width) {
        one[0] += Wide<TD>::one(dy + t * width + col);
        if (last >> e & 1) {
          put_row<TO, 1>(dx + row * width + col, one, scale, accumulate);
          one[0] = 0.f;
        }
      }
    }
  }
}

// A slice of 64 words of one chunk, by a wavefront: the row itself (a row of one chunk) or a partial sum.
template <typename TD, typename TO>
__device__ __forceinline__ void sum_chunk(const TD* dy, const uint32_t* keys, int tile_bits, int64_t width, const Item& item,
                                          const Run* runs, int slice, float scale, bool accumulate, TO* row, float* part) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int first = (int)item.chunk * kChunk;
  const int count = (int)item.tokens - first < kChunk ? (int)item.tokens - first : kChunk;
  // Where this lane's token is: in the last run that starts at or before it.
  const uint32_t want = (uint32_t)(first + (lane < count ? lane : 0));
  uint32_t at = 0, before = 0;
  for (uint32_t r0 = 0; r0 < item.n_runs; r0 += kLanes) {
    const uint32_t r = r0 + lane < item.n_runs ? r0 + lane : item.n_runs - 1;  // the last run again behind the last
    const Run mine = runs[item.first_run + r];
    int found = 0;  // all lanes take part in every exchange, whether or not their run is among these
#pragma unroll
    for (int step = kLanes / 2; step > 0; step >>= 1) {
      const uint32_t start = (uint32_t)__shfl((int)mine.before, found + step, kLanes);
      found += start <= want ? step : 0;
    }
    const uint32_t a = (uint32_t)__shfl((int)mine.at, found, kLanes), b = (uint32_t)__shfl((int)mine.before, found, kLanes);
    at = b <= want ? a : at;
    before = b <= want ? b : before;
  }
  const uint32_t key_at = at + (want - before);
  const int token = (int)((key_at >> tile_bits << tile_bits) + (element(keys, key_at) & ((1u << tile_bits) - 1)));
  const int64_t words = width / kWide;
  const int64_t word = (int64_t)slice * kLanes + lane;
  if ((int64_t)slice * kLanes < words) {
    float acc[1][kWide] = {};
    add_words<TD, 1, kChunkInFlight>(dy, width, word, words, token, count, acc);
    if (word < words) {
      if (part)
        Wide<float>::store(part + word * kWide, acc[0]);
      else
        put_row<TO, kWide>(row + word * kWide, acc[0], scale, accumulate);
    }
  }
  const int64_t col = words * kWide + lane;  // columns behind the last whole word
  if (slice == 0 && words * kWide < width) {
    const float one[1] = {add_singles(dy, width, col, token, count)};
    if (col < width) {
      if (part)
        part[col] = one[0];
      else
        put_row<TO, 1>(row + col, one, scale, accumulate);
    }
  }
}

// The first chunk_blocks workgroups take the chunks, the others the short rows.  A unit of work is a
// wavefront's: a slice of 64 words, so that a wide row's loads are all under way at once rather than
// one slice after the other behind the same look-ups.  (Eight wavefronts to a chunk, joined in LDS,
// spent most of their time on looking up their eight tokens each.)
template <typename TD, typename TO>
__global__ __launch_bounds__(kBlock) void sum_rows(const TD* dy, const uint32_t* keys, int tile_bits, int64_t width,
                                                   float scale, int accumulate, TO* dx, const Taken* taken,
                                                   const uint32_t* entries, const uint32_t* counts, int64_t stride,
                                                   int64_t rows, const Item* singles, const Item* items, const Run* runs,
                                                   float* parts, unsigned chunk_blocks, unsigned slices) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  if (blockIdx.x >= chunk_blocks) {
    const int64_t n_waves = (int64_t)(gridDim.x - chunk_blocks) * kWaves;
    for (int64_t u = (int64_t)(blockIdx.x - chunk_blocks) * kWaves + wave; u < stride * slices; u += n_waves) {
      const int64_t r0 = u / slices;
      sum_short_rows(dy, width, entries, counts, r0, stride, rows, (int)(u - r0 * slices), scale, accumulate != 0, dx);
    }
    return;
  }
  const Taken listed = *taken;
  const uint32_t n_parts = parts_of(listed), n_items = n_parts + singles_of(listed);
  for (uint64_t u = (uint64_t)blockIdx.x * kWaves + wave; u < (uint64_t)n_items * slices; u += (uint64_t)chunk_blocks * kWaves) {
    const uint32_t it = (uint32_t)(u / slices), slice = (uint32_t)(u - (uint64_t)it * slices);
    const Item item = it < n_parts ? items[it] : singles[it - n_parts];
    sum_chunk(dy, keys, tile_bits, width, item, runs, (int)slice, scale, accumulate != 0, dx + (int64_t)item.row * width,
              it < n_parts ? parts + (int64_t)it * width : nullptr);
  }
}

// The chunks of a long row added in order: 64 columns per workgroup, four stretches of chunks.  In fp64, so that a
// row's error is that of its chunks' 32 fp32 additions however many there are (in fp32 a row of 2^22 equal
// tokens was off by 3e-4).
template <typename TO>
__global__ __launch_bounds__(kBlock) void join_chunks(int64_t width, float scale, int accumulate, TO* dx,
                                                     const Taken* taken, const Item* items, const uint32_t* long_rows,
                                                      const float* parts) {
  __shared__ double sums[kWaves][kLanes];
  const int lane = threadIdx.x & (kLanes - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
  const int64_t col = (int64_t)blockIdx.x * kLanes + lane;
  const uint32_t n_long = (uint32_t)taken[1];
  for (uint32_t h = blockIdx.y; h < n_long; h += gridDim.y) {
    const uint32_t it = long_rows[h];  // its first chunk and partial sum
    const Item row = items[it];
    const int chunks = (int)((row.tokens + kChunk - 1) / kChunk);
    const int per = (chunks + kWaves - 1) / kWaves;
    const int from = wave * per, to = from + per < chunks ? from + per : chunks;
    double acc = 0.0;
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
      const float total[1] = {(float)(((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane])};
      put_row<TO, 1>(dx + (int64_t)row.row * width + col, total, scale, accumulate != 0);
    }
  }
}

constexpr int kFewRowsPerWave = 8;
// Eight workgroups per CU; a launch of more would only take longer to start.
constexpr int64_t kMaxFindBlocks = 2048, kMaxSumBlocks = 2048, kMaxFillBlocks = 512;

// Whether the whole gradient is zeroed while the tiles are sorted, which keep few CUs busy, rather than
// the rows without tokens when they are known (us, first and later: 300 tokens over 25128 x 513 rows of
// fp32 24 and 28, 3003 33 and 35, 16384 42.5 and 42.9; over 50257 x 1600 of 16 bits 300 44 and 48, 3003 50
// and 52, 16384 66 and 65, 65536 130 and 118).
bool fill_first(int64_t n, int64_t rows) { return n <= rows / 8; }

template <typename TD, typename TO, typename Id>
void launch_dx(const TD* dy, const Id* ids, int64_t n, const Which& which, int64_t width, float scale, int accumulate,
               TO* dx, char* ws, const Layout& l, hipStream_t s) {
  const int64_t rows = which.rows;
  if (n <= kFewTokens) {
    const int64_t waves = accumulate ? n : (rows + kFewRowsPerWave - 1) / kFewRowsPerWave;
    hipLaunchKernelGGL((few_tokens<TD, TO, Id>), dim3((unsigned)((waves + kWaves - 1) / kWaves)), dim3(kBlock), 0, s, dy, ids,
                       (int)n, which, width, scale, accumulate ? 0 : kFewRowsPerWave, dx);
    return;
  }
  auto* taken = reinterpret_cast<Taken*>(ws + l.taken_at);
  auto* keys = reinterpret_cast<uint32_t*>(ws + l.keys_at);
  auto* index = reinterpret_cast<uint16_t*>(ws + l.index_at);
  auto* entries = reinterpret_cast<uint32_t*>(ws + l.entries_at);
  auto* counts = reinterpret_cast<uint32_t*>(ws + l.counts_at);
  auto* singles = reinterpret_cast<Item*>(ws + l.singles_at);
  auto* items = reinterpret_cast<Item*>(ws + l.items_at);
  auto* long_rows = reinterpret_cast<uint32_t*>(ws + l.long_at);
  auto* runs = reinterpret_cast<Run*>(ws + l.runs_at);
  auto* parts = reinterpret_cast<float*>(ws + l.parts_at);
  const bool fill = !accumulate && fill_first(n, rows);
  const int64_t fill_bytes = fill ? rows * width * (int64_t)sizeof(TO) : 0;
  const int threads = l.tile_bits == kMinTileBits ? kSmallSort : kSort;
  const int64_t fill_blocks = (fill_bytes + threads * 64 - 1) / (threads * 64);
  const unsigned sort_blocks = (unsigned)(l.tiles + (fill_blocks < kMaxFillBlocks ? fill_blocks : kMaxFillBlocks));
  auto sort = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(sort_blocks), dim3(threads), 0, s, ids, n, which, l.tile_bits, l.bucket_bits, l.buckets,
                       keys, index, taken, l.tiles, reinterpret_cast<char*>(dx), fill_bytes);
  };
  switch (l.tile_bits) {
    case kMinTileBits: sort(tile_sort<Id, kSmallSort, 2>); break;
    case 11: sort(tile_sort<Id, kSort, 2>); break;
    case 12: sort(tile_sort<Id, kSort, 4>); break;
    case 13: sort(tile_sort<Id, kSort, 8>); break;
    default: sort(tile_sort<Id, kSort, 16>); break;
  }
  const int group = l.tiles <= kLanes ? kGroup : 1;
  const int64_t max_blocks = ((rows + group - 1) / group + kWaves - 1) / kWaves;
  const unsigned find_blocks = (unsigned)(max_blocks < kMaxFindBlocks ? max_blocks : kMaxFindBlocks);
  auto find = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(find_blocks), dim3(kBlock), 0, s, keys, index, l.tiles, l.tile_bits, l.bucket_bits,
                       l.buckets, rows, width, !accumulate && !fill, dx, taken, entries, counts, singles, items, long_rows, runs);
  };
  if (l.tiles <= 8)
    find(find_rows<TO, kGroup, 1>);
  else if (l.tiles <= 16)
    find(find_rows<TO, kGroup, 2>);
  else if (l.tiles <= 32)
    find(find_rows<TO, kGroup, 4>);
  else if (l.tiles <= kLanes)
    find(find_rows<TO, kGroup, 8>);
  else
    find(find_rows<TO, 1, kMaxTiles / kLanes>);
  const unsigned slices = (unsigned)((width / kWide + kLanes - 1) / kLanes > 0 ? (width / kWide + kLanes - 1) / kLanes : 1);
  const int64_t max_items = (l.max_singles + l.max_parts) * slices;
  const int64_t stride = (rows + kGroup - 1) / kGroup;  // wavefronts with short rows
  const int64_t max_short = (stride * slices + kWaves - 1) / kWaves, max_chunks = (max_items + kWaves - 1) / kWaves;
  const unsigned chunk_blocks = (unsigned)(max_chunks < kMaxSumBlocks ? max_chunks : kMaxSumBlocks);
  const unsigned short_blocks = (unsigned)(max_short < kMaxSumBlocks ? max_short : kMaxSumBlocks);
  hipLaunchKernelGGL((sum_rows<TD, TO>), dim3(chunk_blocks + short_blocks), dim3(kBlock), 0, s, dy, keys, l.tile_bits,
                     width, scale, accumulate, dx, taken, entries, counts, stride, rows, singles, items, runs,
                     parts, chunk_blocks, slices);
  const dim3 join_blocks((unsigned)((width + kLanes - 1) / kLanes), (unsigned)(l.max_long < 128 ? l.max_long : 128));
  hipLaunchKernelGGL(join_chunks<TO>, join_blocks, dim3(kBlock), 0, s, width, scale, accumulate, dx, taken, items, long_rows, parts);
}

int check_common(const char* who, int32_t a_dtype, int32_t b_dtype, int64_t rows, int64_t width, int32_t index_bits, int64_t n,
                 int64_t first_row) {
  if (element_bytes(a_dtype) == 0 || element_bytes(b_dtype) == 0)
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: dtypes %d and %d", who, a_dtype, b_dtype);
  if (index_bits != 32 && index_bits != 64) return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %d-bit indices", who, index_bits);
  if (n < 0 || rows < 0 || width < 0)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: n = %lld, rows = %lld, width = %lld", who, (long long)n, (long long)rows,
                (long long)width);
  if (first_row < 0 || first_row > INT64_MAX - rows)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: first_row = %lld", who, (long long)first_row);
  // Byte offsets stay far inside 63 bits, and the column arithmetic of a workgroup inside 31.
  if (width >= (1LL << 24) || rows >= (1LL << 36) || n >= (1LL << 36))
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %lld rows, %lld tokens of width %lld", who, (long long)rows, (long long)n,
                (long long)width);
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
  const Extent ins[] = {{"x", x, rows * width * element_bytes(x_dtype)}, {"indices", indices, n * (index_bits / 8)}};
  const Extent outs[] = {{"y", y, n * width * element_bytes(y_dtype)}};
  if (int st = check_apart(who, outs, ins)) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {
    with_element(y_dtype, [&](auto ty) {
      using TY = decltype(ty);
      hipLaunchKernelGGL(no_rows<TY>, dim3(1024), dim3(kBlock), 0, s, static_cast<TY*>(y), n * width);
    });
    RAFHIP_HIP_TRY(hipGetLastError());
    return RAFHIP_OK;
  }
  const int words = (int)(width / kWide);
  // Four words in flight per lane where that still leaves every CU several workgroups, one where it does not.
  const int64_t all = n * (words > 0 ? words : 1);
  const int64_t per_block = all >= 256 * 8 * 4 * (int64_t)kBlock ? 4 * kBlock : kBlock;
  int64_t tokens = per_block / (words > 0 ? words : 1);
  tokens = tokens < 1 ? 1 : tokens;
  const int64_t most = kMaxGridBlocks * tokens;  // of a launch
  with_element(x_dtype, [&](auto tx) {
    with_element(y_dtype, [&](auto ty) {
      with_index(index_bits, [&](auto id) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        using Id = decltype(id);
        for (int64_t t0 = 0; t0 < n; t0 += most) {
          const int64_t count = n - t0 < most ? n - t0 : most;
          hipLaunchKernelGGL((embedding_kernel<TX, TY, Id>), dim3((unsigned)((count + tokens - 1) / tokens)), dim3(kBlock), 0, s,
                             static_cast<const TX*>(x), static_cast<const Id*>(indices) + t0, count, rows, first_row, width,
                             words, (int)tokens, scale, static_cast<TY*>(y) + t0 * width);
        }
      });
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}

extern "C" int64_t rafhip_embedding_dx_workspace_bytes(int64_t n, int64_t rows, int64_t width) {
  using namespace rafhip;
  clear_error();
  Layout l;
  if (n < 0 || rows < 0 || width < 0 || width >= (1LL << 24) || !layout_of(n, rows, width, &l)) {
    fail(RAFHIP_ERR_UNSUPPORTED, "rafhip_embedding_dx: %lld tokens over %lld rows of width %lld", (long long)n, (long long)rows,
         (long long)width);
    return -1;
  }
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
  if (need < 0) return RAFHIP_ERR_UNSUPPORTED;  // and the message says why
  if (rows == 0 || width == 0) return RAFHIP_OK;
  if (!dx || (n > 0 && (!dy || !indices))) return fail(RAFHIP_ERR_INVALID_ARG, "%s: null tensor", who);
  if (!is_aligned(dy, element_bytes(dy_dtype)) || !is_aligned(dx, element_bytes(dx_dtype)) || !is_aligned(indices, index_bits / 8))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p of %lld bytes, need %lld", who, workspace, (long long)workspace_bytes,
                (long long)need);
  if (need > 0 && !is_aligned(workspace, 16))
    return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p is not 16-byte aligned", who, workspace);
  if (n == 0 && accumulate) return RAFHIP_OK;
  const Extent ins[] = {{"dy", dy, n * width * element_bytes(dy_dtype)}, {"indices", indices, n * (index_bits / 8)}};
  const Extent outs[] = {{"dx", dx, rows * width * element_bytes(dx_dtype)}, {"workspace", workspace, need}};
  if (int st = check_apart(who, outs, ins)) return st;
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
