// Distillation loss against a teacher's top logits, and its gradient, for gfx950.
//
//   loss = soft T^2 KL(p || softmax(z/T)) + hard CE(label, softmax(z)),  p = softmax over k entries
//   dz   = dloss (soft T (softmax(z/T) - p) + hard (softmax(z) - onehot(label)))
//
// With m = max z and the two sums S_T = sum exp((z-m)/T), S_1 = sum exp(z-m) a row's loss needs its
// k + 1 picked logits only:
//   KL = sum p_j ((t_j - m_t) - (z_j - m))/T - log S_t + log S_T,  CE = log S_1 - (z_label - m),
// and its gradient is an element-wise function of z with k + 1 corrections.  Keeping m and log S
// apart (not their sum) keeps softmax exact to fp32 for logits of any magnitude, rows of the
// type's lowest value included.
//
// What bounds it is memory: n V s bytes to read and, for the gradient, n V s to write.
//   row_loss      forward, a workgroup per row, one pass with a running maximum and sums
//   row_part      the same for few rows: several workgroups per row leave partial sums,
//   join_loss     a wavefront per row joins them
//   row_grad      gradient, workgroups over (row, columns)
//   row_step      both: the row stays in the registers of one workgroup between its sums and its
//                 gradient, so each logit is read once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_table.h"
#include "rafhip_vocab.h"
#include "status.h"
#include "vocab_io.h"

namespace rafhip {
namespace {

constexpr int kLanes = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxTop = RAFHIP_MAX_TOPK;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What the kernels know about a call.
struct Task {
  const void* logits;
  const void* indices;
  const void* teacher;
  const void* labels;
  int64_t rows, row_stride;
  int vocab, topk;
  int teacher_dtype, index_bits;
  float temperature, soft, hard;
  float c_soft;  // log2(e) / T

  // Both without a branch on the type, behind which the compiler would wait for every load: 64 bits or the
  // low half twice, 32 bits or the low half twice.
  __device__ __forceinline__ int64_t index_at(const void* p, int64_t i) const {
    const bool wide = index_bits != 32;
    const RAFHIP_GLOBAL int32_t* at = (const RAFHIP_GLOBAL int32_t*)p + (wide ? 2 * i : i);
    const int32_t low = at[0], high = at[wide ? 1 : 0];
    return wide ? (int64_t)((uint64_t)(uint32_t)high << 32 | (uint32_t)low) : (int64_t)low;
  }
  __device__ __forceinline__ float teacher_at(int64_t i) const {
    const bool wide = teacher_dtype == RAFHIP_F32;
    const RAFHIP_GLOBAL unsigned short* at = (const RAFHIP_GLOBAL unsigned short*)teacher + (wide ? 2 * i : i);
    const unsigned short low = at[0], high = at[wide ? 1 : 0];
    const float half = (float)__builtin_bit_cast(_Float16, low);
    const float other = __uint_as_float(wide ? (uint32_t)high << 16 | low : (uint32_t)low << 16);
    return teacher_dtype == RAFHIP_F16 ? half : other;
  }
  // Column of teacher entry j of a row, -1 if it is absent; *t is its logit.
  __device__ __forceinline__ int entry(int64_t row, int j, float* t) const {
    const int64_t i = index_at(indices, row * topk + j);
    *t = teacher_at(row * topk + j);
    return i >= 0 && i < vocab && *t != -INFINITY ? (int)i : -1;
  }
  __device__ __forceinline__ int label(int64_t row) const {
    if (!labels) return -1;
    const int64_t i = index_at(labels, row);
    return i >= 0 && i < vocab ? (int)i : -1;
  }
};

template <typename F>
__device__ __forceinline__ float wave_reduce(float x, F&& f) {
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) x = f(x, __shfl_xor(x, d, kLanes));
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
  return wave_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_add(float x) {
  return wave_reduce(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ double wave_add(double x) {
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) x += __shfl_xor(x, d, kLanes);
  return x;
}

// The teacher's softmax of one row, computed by a whole wavefront: p_j = exp2((t_j - top) c) / sum.
struct Teacher {
  float top, sum;
  bool any;
};
__device__ __forceinline__ Teacher teacher_of(const Task& a, int64_t row) {
  constexpr int kHeld = 2;  // entries of a lane that are requested at once, and kept where there are no more
  const int lane = threadIdx.x & (kLanes - 1);
  Teacher r;
  float held[kHeld];
  float top = -INFINITY;
  bool any = false;
  auto request = [&](int j0) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int j = j0 + u * kLanes + lane;
      const int at = a.entry(row, j < a.topk ? j : a.topk - 1, &held[u]);
      if (j >= a.topk || at < 0) held[u] = -INFINITY;  // as an entry that is absent
      any |= j < a.topk && at >= 0;
    }
  };
  for (int j0 = 0; j0 < a.topk; j0 += kHeld * kLanes) {
    request(j0);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) top = fmaxf(top, held[u]);
  }
  r.any = __any(any);
  r.top = wave_max(top);
  float sum = 0.f;
  for (int j0 = 0; j0 < a.topk; j0 += kHeld * kLanes) {
    if (a.topk > kHeld * kLanes) request(j0);
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (held[u] != -INFINITY) sum += exp2_hw((held[u] - r.top) * a.c_soft);
  }
  r.sum = wave_add(sum);
  return r;
}

// Whether a row has any teacher entry, found by a wavefront (the same in all lanes): one round trip
// where the first 64 have one, before anything else of the row is read.
__device__ __forceinline__ bool any_entry(const Task& a, int64_t row) {
  const int lane = threadIdx.x & (kLanes - 1);
  for (int j0 = 0; j0 < a.topk; j0 += kLanes) {
    float t;
    if (__any(j0 + lane < a.topk && a.entry(row, j0 + lane, &t) >= 0)) return true;
  }
  return false;
}

// Which sums a row needs.  kOne: a single factor serves whatever is wanted -- T == 1, or only one of the
// two terms.  Else both exp((z - m)/T) and exp(z - m); for the temperatures 2 and 4 the second is a
// power of the first, which saves an exponential (a quarter-rate instruction) per element and pass:
// of 8192 rows of 50257 in 16 bits the loss takes 144 us with the square and 166 with two exponentials,
// the gradient 308 and 320, both at once 354 and 383.
enum { kOne = 0, kBoth, kSquare, kFourth };

// Maximum and sums over the columns a lane has seen.  c0 is log2(e)/T, or log2(e) if only the
// hard term is wanted.
template <int kSums>
struct Exps {
  float m = -INFINITY;
  float s0 = 0.f, s1 = 0.f;

  // A maximum of -inf stands for "nothing yet": exponents are then taken against zero, so that
  // -inf - -inf does not arise.
  static __device__ __forceinline__ float base(float m) { return m == -INFINITY ? 0.f : m; }

  // exp(d) where e = exp(d / T).
  static __device__ __forceinline__ float hard(float d, float e) {
    if constexpr (kSums == kSquare) return e * e;
    if constexpr (kSums == kFourth) return (e * e) * (e * e);
    return exp2_hw(d * kLog2e);
  }

  __device__ __forceinline__ void rescale(float m2, float c0) {
    const float d = m - base(m2), e = exp2_hw(d * c0);
    s0 *= e;
    if constexpr (kSums != kOne) s1 *= hard(d, e);
    m = m2;
  }
  __device__ __forceinline__ void term(float z, float b, float c0) {
    const float d = z - b, e = exp2_hw(d * c0);
    s0 += e;
    if constexpr (kSums != kOne) s1 += hard(d, e);
  }
  __device__ __forceinline__ void merge(float om, float o0, float o1, float c0) {
    rescale(fmaxf(m, om), c0);
    const float d = om - base(m), e = exp2_hw(d * c0);
    s0 += o0 * e;
    if constexpr (kSums != kOne) s1 += o1 * hard(d, e);
  }
  __device__ __forceinline__ void wave_merge(float c0) {
    rescale(wave_max(m), c0);
    s0 = wave_add(s0);
    if constexpr (kSums != kOne) s1 = wave_add(s1);
  }
};

// Joined over the workgroup, the same in every thread; `red` holds three floats per wavefront.
template <int kSums>
__device__ __forceinline__ void block_merge(Exps<kSums>& a, float (*red)[3], float c0) {
  a.wave_merge(c0);
  if ((threadIdx.x & (kLanes - 1)) == 0) {
    float* r = red[threadIdx.x / kLanes];
    r[0] = a.m;
    r[1] = a.s0;
    r[2] = a.s1;
  }
  __syncthreads();
  Exps<kSums> all;
  const int waves = (int)blockDim.x / kLanes;
  for (int w = 0; w < waves; ++w) all.merge(red[w][0], red[w][1], red[w][2], c0);
  a = all;
}

// A stretch of columns as up to `head` single elements, whole words and a tail: 16-bit rows of an
// odd width start at an odd multiple of two bytes every other row, and words there would cost a
// quarter of the bandwidth.
struct Stretch {
  int head, words, tail_at, tail;
};
template <typename T>
__device__ __forceinline__ Stretch stretch_of(const T* at, int count) {
  Stretch s;
  s.head = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(at) & 2) && count > 0 ? 1 : 0;
  s.words = (count - s.head) / kWide;
  s.tail_at = s.head + s.words * kWide;
  s.tail = count - s.tail_at;
  return s;
}

// The sums over `count` columns at z, by the workgroup.  With kLong a thread adds the 32 columns that it has in
// flight in fp32 and these sums in fp64: in fp32 throughout, each of the thousands of columns that a
// thread has of a long row would be rounded to the step of the sum so far (65 rows of 2^24 columns: log S
// off by 2e-4).
template <typename T, int kSums, bool kLong>
__device__ __forceinline__ void add_columns(Exps<kSums>& a, const T* z, int count, float c0) {
  constexpr int kInFlight = 4;
  const int block = (int)blockDim.x;
  const Stretch s = stretch_of(z, count);
  double s0 = 0.0, s1 = 0.0;  // relative to a.m
  for (int w0 = threadIdx.x; w0 < s.words; w0 += block * kInFlight) {
    typename Wide<T>::Raw raw[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      // Without a condition, the last word again behind the last: the compiler puts a wait for all
      // earlier loads in front of every load in a branch.
      const int w = w0 + u * block < s.words ? w0 + u * block : s.words - 1;
      raw[u] = Wide<T>::load(z + s.head + (int64_t)w * kWide);
    }
    float top = a.m;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
#pragma unroll
      for (int j = 0; j < kWide; ++j) top = fmaxf(top, Wide<T>::get(raw[u], j));
    }
    const float b = Exps<kSums>::base(top);
    if constexpr (kLong) {
      const float d = a.m - b, e = exp2_hw(d * c0);
      s0 *= e;
      if constexpr (kSums != kOne) s1 *= Exps<kSums>::hard(d, e);
      a.m = top;
      a.s0 = a.s1 = 0.f;
    } else {
      a.rescale(top, c0);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (w0 + u * block < s.words) {
#pragma unroll
        for (int j = 0; j < kWide; ++j) a.term(Wide<T>::get(raw[u], j), b, c0);
      }
    }
    if constexpr (kLong) {
      s0 += a.s0;
      if constexpr (kSums != kOne) s1 += a.s1;
    }
  }
  if constexpr (kLong) {
    a.s0 = (float)s0;
    a.s1 = (float)s1;
  }
  // The single elements: the first and the last few, one per thread.
  const int i = (int)threadIdx.x;
  if (i < s.head + s.tail) {
    const float x = Wide<T>::one(z + (i < s.head ? i : s.tail_at + i - s.head));
    a.rescale(fmaxf(a.m, x), c0);
    a.term(x, Exps<kSums>::base(a.m), c0);
  }
}

// Which sums a row's loss needs, and what they are called.
struct RowSums {
  float m;
  double log_soft, log_hard;  // log S_T, log S_1
};
template <int kSums>
__device__ __forceinline__ RowSums row_sums_of(const Exps<kSums>& s) {
  RowSums r;
  r.m = s.s0 != s.s0 && s.m != INFINITY ? NAN : s.m;  // the running maximum passes over a NaN
  r.log_soft = s.m == -INFINITY ? (double)NAN : log((double)s.s0);  // nothing but -inf has no softmax
  r.log_hard = kSums != kOne && s.m != -INFINITY ? log((double)s.s1) : r.log_soft;
  return r;
}

// Loss and stats of a row, by one wavefront.
template <typename T>
__device__ __forceinline__ void finish_row(const Task& a, int64_t row, const Teacher& t, int label, const RowSums& s,
                                           float* loss, float* stats) {
  const int lane = threadIdx.x & (kLanes - 1);
  const T* z = (const T*)a.logits + row * a.row_stride;
  const double inv_t = 1.0 / (double)a.temperature;
  double value = 0.0;
  if (t.any) {
    double cross = 0.0;  // sum of A_j ((t_j - top) - (z_j - m)), A_j = p_j * sum
    for (int j = lane; j < a.topk; j += kLanes) {
      float tj;
      const int at = a.entry(row, j, &tj);
      if (at >= 0) {
        const float w = exp2_hw((tj - t.top) * a.c_soft);
        if (w != 0.f) cross += (double)w * (((double)tj - (double)t.top) - ((double)Wide<T>::one(z + at) - (double)s.m));
      }
    }
    cross = wave_add(cross);
    const double kl = cross * inv_t / (double)t.sum - log((double)t.sum) + s.log_soft;
    value += (double)a.soft * (double)a.temperature * (double)a.temperature * kl;
  }
  if (label >= 0) value += (double)a.hard * (s.log_hard - ((double)Wide<T>::one(z + label) - (double)s.m));
  if (lane == 0) {
    loss[row] = (float)value;
    if (stats) {
      const bool some = t.any || label >= 0;
      stats[row * 3] = some ? s.m : 0.f;
      stats[row * 3 + 1] = t.any ? (float)s.log_soft : 0.f;
      stats[row * 3 + 2] = label >= 0 ? (float)s.log_hard : 0.f;
    }
  }
}

constexpr int kMaxBlock = 1024;

template <typename T, int kSums, bool kLong>
__global__ __launch_bounds__(kMaxBlock, kLong ? 7 : 8) void row_loss(Task a, float c0, float* loss, float* stats) {
  __shared__ float red[kMaxBlock / kLanes][3];
  const int64_t row = blockIdx.x;
  const Teacher t = teacher_of(a, row);
  const int label = a.label(row);
  Exps<kSums> s;
  if (t.any || label >= 0) {  // the same in all threads
    add_columns<T, kSums, kLong>(s, (const T*)a.logits + row * a.row_stride, a.vocab, c0);
    block_merge(s, red, c0);
  }
  if (threadIdx.x < kLanes) finish_row<T>(a, row, t, label, row_sums_of(s), loss, stats);
}

constexpr int kPartBlock = 256;

// Columns [split * per_split, ...) of a row: partial sums to parts[row][split][4].
template <typename T, int kSums>
__global__ __launch_bounds__(kPartBlock) void row_part(Task a, float c0, int per_split, float* parts) {
  __shared__ float red[kPartBlock / kLanes][3];
  const int64_t row = blockIdx.y;
  const int from = (int)blockIdx.x * per_split;
  const int count = a.vocab - from < per_split ? a.vocab - from : per_split;
  Exps<kSums> s;
  if (a.label(row) >= 0 || any_entry(a, row)) {  // a row without targets is not read
    add_columns<T, kSums, false>(s, (const T*)a.logits + row * a.row_stride + from, count, c0);
    block_merge(s, red, c0);
  }
  if (threadIdx.x == 0) {
    float* p = parts + (row * gridDim.x + blockIdx.x) * 4;
    p[0] = s.m;
    p[1] = s.s0;
    p[2] = s.s1;
  }
}

// The sums of a row from its parts, by a wavefront (the same in all lanes).
template <int kSums>
__device__ __forceinline__ Exps<kSums> join_parts(const float* parts, int64_t row, int splits, float c0) {
  Exps<kSums> s;
  const int lane = threadIdx.x & (kLanes - 1);
  for (int i = lane; i < splits; i += kLanes) {
    const float* p = parts + (row * splits + i) * 4;
    s.merge(p[0], p[1], p[2], c0);
  }
  s.wave_merge(c0);
  return s;
}

template <typename T, int kSums>
__global__ __launch_bounds__(kLanes) void join_loss(Task a, float c0, const float* parts, int splits, float* loss,
                                                    float* stats) {
  const int64_t row = blockIdx.x;
  const Teacher t = teacher_of(a, row);
  finish_row<T>(a, row, t, a.label(row), row_sums_of(join_parts<kSums>(parts, row, splits, c0)), loss, stats);
}

// ------------------------------------------------------------------------------------ gradient
// g(z) = a0 exp2((z - m) c0 - l0) [+ a1 exp2((z - m) log2(e) - l1)], before the corrections.  Where the
// second exponential is a power of the first, l0 is taken so that this power is the label's softmax
// itself, and a0 makes up for it.  That factor is at most 1, since S_1 is at most the power of S_T (the other way round
// a1 would have to hold up to vocab^3, beyond fp32 for large dloss).
struct Grad {
  float m, c0, l0, a0, l1, a1;
  template <int kSums>
  __device__ __forceinline__ float at(float z) const {
    const float d = z - m, e = exp2_hw(fmaf(d, c0, -l0));
    if constexpr (kSums == kSquare) return e * fmaf(a1, e, a0);
    if constexpr (kSums == kFourth) return e * fmaf(a1 * e, e * e, a0);
    if constexpr (kSums == kBoth) return fmaf(a1, exp2_hw(fmaf(d, kLog2e, -l1)), a0 * e);
    return a0 * e;
  }
};

template <int kSums>
__device__ __forceinline__ Grad grad_of(const Task& a, float c0, float dloss, bool soft, bool hard, float m, float log2_soft,
                                        float log2_hard) {
  Grad g;
  const float as = soft ? dloss * a.soft * a.temperature : 0.f, ah = hard ? dloss * a.hard : 0.f;
  g.m = m;
  g.c0 = c0;
  if constexpr (kSums != kOne) {
    g.l0 = log2_soft;
    g.a0 = as;
    g.l1 = log2_hard;
    g.a1 = ah;
    if constexpr (kSums == kSquare || kSums == kFourth) {
      g.l0 = (kSums == kSquare ? 0.5f : 0.25f) * log2_hard;
      g.a0 = soft ? as * exp2_hw(g.l0 - log2_soft) : 0.f;
    }
  } else {
    g.l0 = soft ? log2_soft : log2_hard;
    g.a0 = as + ah;
    g.l1 = g.a1 = 0.f;
  }
  return g;
}

template <int kSums>
__device__ __forceinline__ Grad grad_of(const Task& a, float c0, float dloss, bool soft, bool hard, const Exps<kSums>& s) {
  const float log2_soft = s.m == -INFINITY ? NAN : __builtin_amdgcn_logf(s.s0);  // base 2
  return grad_of<kSums>(a, c0, dloss, soft, hard, s.m, log2_soft, kSums != kOne ? __builtin_amdgcn_logf(s.s1) : log2_soft);
}

// The columns a row's targets correct, the label last.  Teacher entries with the same column are taken
// together by the first of them; whether there are any is found by a hash table, since comparing all
// pairs would cost more than the row for hundreds of entries.  The label, which is among the teacher's
// entries more often than not, is only looked up there.
// In dynamic LDS: picks_bytes(topk) bytes.
struct Picks {
  int n, n_slots;  // topk and the label; a power of two of at least twice that many
  int* at;
  float* minus;
  int* slots;
  int* twice;

  __device__ __forceinline__ Picks(int topk, int log2_slots, int* lds) {
    n = topk + 1;
    n_slots = 1 << log2_slots;
    twice = lds;
    at = lds + 1;
    minus = (float*)(at + n);
    slots = (int*)(minus + n);
  }
};
inline int picks_log2_slots(int topk) {
  int log2 = 5;
  while ((1 << log2) < 2 * (topk + 1)) ++log2;
  return log2;
}
inline size_t picks_bytes(int topk) {
  return 4 * (1 + 2 * ((size_t)topk + 1) + ((size_t)1 << picks_log2_slots(topk)));
}

// In steps: empty the table; list the targets of a row that lie in [from, from + count); enter them into
// the table, behind a barrier after the first step; put_picks, behind another after all.
__device__ __forceinline__ void clear_picks(const Picks& p) {
  for (int i = threadIdx.x; i < p.n_slots; i += (int)blockDim.x) p.slots[i] = -1;
  if (threadIdx.x == 0) *p.twice = 0;
}

__device__ __forceinline__ void list_picks(const Task& a, int64_t row, const Teacher& t, int label, float dloss, int from,
                                           int count, const Picks& p) {
  const float scale = dloss * a.soft * a.temperature;
  for (int j = threadIdx.x; j < p.n; j += (int)blockDim.x) {
    int at = -1;
    float minus = 0.f;
    if (j == a.topk) {
      at = label;
      minus = dloss * a.hard;
    } else {
      float tj;
      at = a.entry(row, j, &tj);
      minus = scale * (exp2_hw((tj - t.top) * a.c_soft) / t.sum);
    }
    at = at >= from && at < from + count ? at : -1;
    p.at[j] = at;
    p.minus[j] = minus;
  }
}

// Each thread enters the teacher's entries that it has listed.
__device__ __forceinline__ void enter_picks(const Picks& p) {
  for (int j = threadIdx.x; j < p.n - 1; j += (int)blockDim.x) {
    const int at = p.at[j];
    if (at < 0) continue;
    for (int h = at & (p.n_slots - 1);; h = (h + 1) & (p.n_slots - 1)) {  // half of the slots stay free
      const int before = atomicCAS(&p.slots[h], -1, at);
      if (before == -1) break;
      if (before == at) {
        *p.twice = 1;
        break;
      }
    }
  }
}

template <typename T, int kSums>
__device__ __forceinline__ void put_picks(const Picks& p, const Grad& g, const T* z, T* out) {
  const bool twice = *p.twice != 0;
  const int label = p.at[p.n - 1];
  for (int j = threadIdx.x; j < p.n; j += (int)blockDim.x) {
    const int at = p.at[j];
    if (at < 0) continue;
    float minus = p.minus[j];
    if (twice) {
      bool first = true;
      for (int i = 0; i < j && first; ++i) first = p.at[i] != at;
      if (!first) continue;
      for (int i = j + 1; i < p.n; ++i)
        if (p.at[i] == at) minus += p.minus[i];
    } else if (j < p.n - 1) {
      if (at == label) minus += p.minus[p.n - 1];
    } else {
      int h = at & (p.n_slots - 1);
      while (p.slots[h] != -1 && p.slots[h] != at) h = (h + 1) & (p.n_slots - 1);
      if (p.slots[h] == at) continue;  // its part is that entry's
    }
    Wide<T>::put(out + at, g.template at<kSums>(Wide<T>::one(z + at)) - minus);
  }
}

template <typename T>
__device__ __forceinline__ void put_zeros(T* out, int64_t count) {
  const float none[kWide] = {};
  const int64_t words = count / kWide;
  for (int64_t w = threadIdx.x; w < words; w += (int)blockDim.x) Wide<T>::store(out + w * kWide, none);
  for (int64_t i = words * kWide + threadIdx.x; i < count; i += (int)blockDim.x) Wide<T>::put(out + i, 0.f);
}

constexpr int kGradBlock = 256;

// Columns [split * per_split, ...) of a row.  With `parts` the row's sums are joined from them and one more
// workgroup, without columns, writes the loss; otherwise they come from `stats`.
template <typename T, int kSums>
__global__ __launch_bounds__(kGradBlock) void row_grad(Task a, float c0, int per_split, const float* dloss, int dloss_step,
                                                       const float* stats, const float* parts, int n_parts, float* loss,
                                                       T* dlogits, int64_t out_width, int log2_slots) {
  constexpr int kInFlight = 4;
  extern __shared__ int lds[];
  const Picks picks(a.topk, log2_slots, lds);
  const int64_t row = blockIdx.y;
  const int from = (int)blockIdx.x * per_split;
  const int count = a.vocab - from < per_split ? a.vocab - from : per_split;
  const int label = a.label(row);
  const float dl = dloss[row * dloss_step];
  T* out_row = dlogits + row * out_width;
  const T* z_row = (const T*)a.logits + row * a.row_stride;
  const T* z = z_row + from;
  T* out = out_row + from;
  if (blockIdx.x == gridDim.x - 1) put_zeros<T>(out_row + a.vocab, out_width - a.vocab);
  if (count <= 0 && !parts) return;  // a vocabulary without columns: its padding is all there is
  const Teacher t = teacher_of(a, row);
  if (count <= 0) {  // the workgroup of the loss
    if (threadIdx.x < kLanes)
      finish_row<T>(a, row, t, label, row_sums_of(join_parts<kSums>(parts, row, n_parts, c0)), loss, nullptr);
    return;
  }
  if (!t.any && label < 0) return put_zeros<T>(out, count);
  const Stretch s = stretch_of(out, count);
  typename Wide<T>::Raw raw[kInFlight];
  auto request = [&](int w0) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int w = w0 + u * kGradBlock < s.words ? w0 + u * kGradBlock : s.words - 1;
      raw[u] = Wide<T>::load(z + s.head + (int64_t)w * kWide);
    }
  };
  if (s.words > 0) request(threadIdx.x);
  clear_picks(picks);
  list_picks(a, row, t, label, dl, from, count, picks);
  __syncthreads();
  enter_picks(picks);
  Grad g;
  if (parts) {
    const Exps<kSums> sums = join_parts<kSums>(parts, row, n_parts, c0);
    g = grad_of<kSums>(a, c0, dl, t.any, label >= 0, sums);
  } else {
    g = grad_of<kSums>(a, c0, dl, t.any, label >= 0, stats[row * 3], stats[row * 3 + 1] * kLog2e, stats[row * 3 + 2] * kLog2e);
  }
  for (int w0 = threadIdx.x; w0 < s.words; w0 += kGradBlock * kInFlight) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int w = w0 + u * kGradBlock;
      if (w < s.words) {
        float v[kWide];
#pragma unroll
        for (int j = 0; j < kWide; ++j) v[j] = g.template at<kSums>(Wide<T>::get(raw[u], j));
        Wide<T>::store(out + s.head + (int64_t)w * kWide, v);
      }
    }
    if (w0 + kGradBlock * kInFlight < s.words) request(w0 + kGradBlock * kInFlight);
  }
  const int i = (int)threadIdx.x;
  if (i < s.head + s.tail) {
    const int c = i < s.head ? i : s.tail_at + i - s.head;
    Wide<T>::put(out + c, g.template at<kSums>(Wide<T>::one(z + c)));
  }
  __syncthreads();
  put_picks<T, kSums>(picks, g, z_row, out_row);
}

// Words of a thread for which there are kernels; the first of a kernel's words that may not exist.
template <typename T>
struct StepWords;
template <>
struct StepWords<float> {
  static constexpr int kCount = 6, kList[kCount] = {1, 2, 4, 6, 9, 12};
};
template <>
struct StepWords<_Float16> {
  static constexpr int kCount = 8, kList[kCount] = {1, 2, 4, 8, 12, 16, 20, 25};
};
template <>
struct StepWords<Bf16> : StepWords<_Float16> {};

// Loss and gradient of a row whose words stay in the registers of a workgroup, kWords a thread, so that
// each logit is read once.  With many rows the workgroup is the smallest that holds a row: four of 256
// threads share a CU, and while one waits for its row or for the others' sums the rest read, compute
// and write (8192 rows of 50257 in 16 bits, T = 2 with labels: 354 us, with one of 1024 threads 461;
// T = 1 without labels 350 both).  The most words per thread do not quite fit beside the rest: of the variants
// of 25 words the compiler keeps 3 registers in scratch with one sum, 13 at T = 2 and 4, 22 (bf16) or 40 (fp16) at other
// temperatures with labels, and of those of 12 fp32 words 6 to 8 with two sums; no other variant has any.
template <typename T, int kSums, int kWords, int kSure>
__global__ __launch_bounds__(kMaxBlock, 4) void row_step(Task a, float c0, const float* dloss, int dloss_step, float* loss,
                                                            T* dlogits, int64_t out_width, int log2_slots) {
  __shared__ float red[2][kMaxBlock / kLanes][2];
  extern __shared__ int lds[];
  const Picks picks(a.topk, log2_slots, lds);
  const int block = (int)blockDim.x, waves = block / kLanes;
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.logits + row * a.row_stride;
  T* out = dlogits + row * out_width;
  const Stretch s = stretch_of(out, a.vocab);
  const int i = (int)threadIdx.x;
  const bool single = i < s.head + s.tail;
  const int single_at = i < s.head ? i : s.tail_at + i - s.head;
  const int label = a.label(row);
  const float dl = dloss[row * dloss_step];
  put_zeros<T>(out + a.vocab, out_width - a.vocab);
  const Teacher t = teacher_of(a, row);
  if (!t.any && label < 0) {
    put_zeros<T>(out, a.vocab);
    if (i == 0) loss[row] = 0.f;
    return;
  }
  // Word u of a thread lies a fixed distance behind word 0, so one register of offset serves them all.
  auto exists = [&](int u) { return u < kSure || i + u * block < s.words; };
  const uint32_t off = (uint32_t)i * (kWide * sizeof(T));
  const T* z0 = z + s.head;
  T* out0 = out + s.head;
  auto word_of = [&](const T* base, int u) { return (const T*)((const char*)(base + u * block * kWide) + off); };
  typename Wide<T>::Raw raw[kWords];
  if (s.words > 0) {
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const int w = i + u * block;
      raw[u] = Wide<T>::load(u < kSure ? word_of(z0, u) : z0 + (int64_t)(w < s.words ? w : s.words - 1) * kWide);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kWords; ++u) raw[u] = Wide<T>::fill(-INFINITY);
  }
  const float x1 = single ? Wide<T>::one(z + single_at) : -INFINITY;
  clear_picks(picks);
  // The row's maximum first: the sums then need no rescaling.
  float top = x1;
#pragma unroll
  for (int u = 0; u < kWords; ++u) {
#pragma unroll
    for (int j = 0; j < kWide; ++j) top = fmaxf(top, Wide<T>::get(raw[u], j));
  }
  top = wave_max(top);
  if ((i & (kLanes - 1)) == 0) red[0][i / kLanes][0] = top;
  __syncthreads();
  for (int w = 0; w < waves; ++w) top = fmaxf(top, red[0][w][0]);
  // The words are widened again for the sums and for the gradient: as fp32 numbers the row would not
  // fit.
#pragma unroll
  for (int u = 0; u < kWords; ++u) Wide<T>::keep_narrow(raw[u]);
  Exps<kSums> sums;
  sums.m = top;
  const float b = Exps<kSums>::base(top);
#pragma unroll
  for (int u = 0; u < kWords; ++u) {
    if (exists(u)) {
#pragma unroll
      for (int j = 0; j < kWide; ++j) sums.term(Wide<T>::get(raw[u], j), b, c0);
    }
  }
  if (single) sums.term(x1, b, c0);
  sums.s0 = wave_add(sums.s0);
  if constexpr (kSums != kOne) sums.s1 = wave_add(sums.s1);
  if ((i & (kLanes - 1)) == 0) {
    red[1][i / kLanes][0] = sums.s0;
    red[1][i / kLanes][1] = sums.s1;
  }
  __syncthreads();
  sums.s0 = sums.s1 = 0.f;
  for (int w = 0; w < waves; ++w) {
    sums.s0 += red[1][w][0];
    sums.s1 += red[1][w][1];
  }
#pragma unroll
  for (int u = 0; u < kWords; ++u) Wide<T>::keep_narrow(raw[u]);
  const Grad g = grad_of<kSums>(a, c0, dl, t.any, label >= 0, sums);
#pragma unroll
  for (int u = 0; u < kWords; ++u) {
    if (exists(u)) {
      float v[kWide];
#pragma unroll
      for (int j = 0; j < kWide; ++j) v[j] = g.template at<kSums>(Wide<T>::get(raw[u], j));
      Wide<T>::store(const_cast<T*>(word_of(out0, u)), v);
    }
  }
  if (single) Wide<T>::put(out + single_at, g.template at<kSums>(x1));
  if (i < kLanes) finish_row<T>(a, row, t, label, row_sums_of(sums), loss, nullptr);
  list_picks(a, row, t, label, dl, 0, a.vocab, picks);  // now that the row's registers are free
  enter_picks(picks);
  __syncthreads();
  put_picks<T, kSums>(picks, g, z, out);
}

// ---------------------------------------------------------------------------------------- host
constexpr int64_t kManyRows = 512;  // rows that keep the GPU busy with a workgroup of 256 threads each
constexpr int64_t kFewRows = 64;    // rows that leave most CUs idle with one workgroup each
constexpr int kWantBlocks = 1024;   // four workgroups for each of 256 CUs
constexpr int kMinPerSplit = 4096;    // columns below which another workgroup does not pay
constexpr int kGradColumns = 8192;    // of a row_grad workgroup: four words a thread, requested at once
constexpr int kPartColumns = 32768;   // of a row_part workgroup at most

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Columns per workgroup so that `rows` rows make kWantBlocks workgroups, a multiple of a word.
int columns_per_split(int64_t rows, int64_t vocab, int64_t most) {
  int64_t per = ceil_div(vocab, ceil_div(kWantBlocks, rows < 1 ? 1 : rows));
  if (per > most) per = ceil_div(vocab, ceil_div(vocab, most));
  if (per < kMinPerSplit) per = kMinPerSplit;
  return (int)((per + kWide - 1) / kWide * kWide);
}

// The forward call.  A few long rows are read by several workgroups each, whose partial sums a second
// launch joins.  Columns count rather than bytes, since a thread waits for its chain of exponentials as much as
// for its words (T = 2 with labels, us whole and split: 8 rows of 50257 8.6 and 8.1 in fp32, 8.5 and 8.1 in 16 bits,
// of 160000 15.2 and 8.3, 15.1 and 8.2; 64 rows of 50257 8.7 and 9.4, 8.5 and 9.3, of 65536 9.6 and 9.4, 9.4 and
// 9.2, of 160000 17.5 and 14.1, 15.2 and 11.5; 256 rows of 160000 29.6 and 31.4, 19 and 22).  Between 64 and
// 256 rows the two cross, in 16 bits later than in fp32, and the rule leaves up to a quarter there (65 rows of
// 160000 17.5 and 14.3, 15.2 and 11.7; 100 rows 18.2 and 18.4, 16.7 and 13.7; 150 rows 20.2 and 22.6, 18.2 both).
bool loss_is_split(int64_t rows, int64_t vocab) { return rows <= kFewRows && vocab > 65536; }

// Otherwise a workgroup reads a row, a larger one where there are not many and they are long (16 bits, us
// with 256 and 512 threads: 256 rows of 8192 5.6 and 6.5; 8 rows of 50257 9.2 and 8.3, 256 11.5 and 10.0).
int loss_block(int64_t rows, int64_t vocab) { return rows < kManyRows && vocab > 16384 ? 512 : 256; }

// Columns of a thread whose sum fp32 takes one after the other; row_part's threads have 128 at most, row_step's
// 200.  Rows beyond pay for the fp64 sums (16 bits, us without and with: 2048 rows of 131072 97.3 and 97.2 at T = 1,
// 103.1 and 104 at T = 1.5 with labels, 100.4 and 105.9 at T = 4; 4096 rows of 50257 at T = 4 80 and 85).
constexpr int kMaxChain = 224;

// Threads of row_step for a row, the fewest whose registers hold it, from 256 with many rows and from 512
// with fewer, or 0: then row_part and row_grad read it twice, with workgroups for every CU.  So are a few
// long rows (T = 2 with labels, us once and twice: 8 rows of 16384 8.2 and 8.5 in fp32, 8.4 both in 16 bits, of 32000
// 10.7 and 8.8, 10 and 8.6, of 98000 18.4 and 8.9, 17.4 and 8.7; 64 rows of 16384 12.9 and 12.5, 12.7 and 12.9, of 32000
// 15.7 and 14, 14.2 and 12.2, of 98000 25.8 and 21.7, 19.5 and 14.9; but 256 rows of 50257 28.5 and 34.4, 20.7 and 25;
// 2048 of 98000 in fp32 395 and 442, of 200000 in 16 bits 436 and 468).  From 65 to about 100 rows twice is still the
// faster of the two for long ones (65 rows of 98000 23.3 and 21.6, 19.8 and 15.1; 100 rows 28.7 and 30.2, 23.5 and
// 21), and so it is for the longest at other temperatures with labels, whose words spill (2048 of 200000 at
// T = 1.5 496 and 480 in bf16, 516 and 485 in fp16).
template <typename T>
int block_for_row(int64_t rows, int64_t vocab) {
  if (rows <= kFewRows && vocab > 24576) return 0;
  for (int block = rows < kManyRows ? 512 : 256; block <= kMaxBlock; block *= 2)
    if (vocab / kWide <= (int64_t)block * StepWords<T>::kList[StepWords<T>::kCount - 1]) return block;
  return 0;
}
int step_block(int64_t rows, int64_t vocab, int32_t dtype) {
  return dtype == RAFHIP_F32 ? block_for_row<float>(rows, vocab) : block_for_row<_Float16>(rows, vocab);
}

int64_t parts_bytes(int64_t rows, int64_t vocab) {
  return rows * ceil_div(vocab, columns_per_split(rows, vocab, kPartColumns)) * 16;
}

// Calls f with the kernel for `words` words a thread: the next larger of the list.  All words that the
// kernel before it has exist in every thread, whether or not the row starts with a single element:
// a row has vocab / kWide words or one less, and vocab / kWide exceeds theirs by one at least.
template <typename T, int kSums, int kAt = 0, typename F>
void with_step_kernel(int words, F&& f) {
  constexpr int kWords = StepWords<T>::kList[kAt], kSure = kAt > 0 ? StepWords<T>::kList[kAt > 0 ? kAt - 1 : 0] : 0;
  if constexpr (kAt + 1 < StepWords<T>::kCount) {
    if (words > kWords) return with_step_kernel<T, kSums, kAt + 1>(words, f);
  }
  f(row_step<T, kSums, kWords, kSure>);
}

int check_args(const char* who, const rafhip_topk_distill_args* p) {
  if (!p) return fail(RAFHIP_ERR_INVALID_ARG, "%s: args is NULL", who);
  const rafhip_topk_distill_args& a = *p;
  if (element_bytes(a.logits_dtype) == 0 || element_bytes(a.topk_dtype) == 0)
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: dtypes %d and %d", who, a.logits_dtype, a.topk_dtype);
  if (a.index_bits != 32 && a.index_bits != 64) return fail(RAFHIP_ERR_UNSUPPORTED, "%s: %d-bit indices", who, a.index_bits);
  if (a.rows < 0 || a.vocab < 0 || a.topk < 0 || a.row_stride < a.vocab)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: rows = %lld, vocab = %lld, row_stride = %lld, topk = %d", who, (long long)a.rows,
                (long long)a.vocab, (long long)a.row_stride, a.topk);
  if (a.vocab >= (1LL << 28) || a.row_stride >= (1LL << 28) || a.rows >= (1LL << 31) || a.topk > kMaxTop)
    return fail(RAFHIP_ERR_UNSUPPORTED, "%s: rows = %lld, vocab = %lld, row_stride = %lld, topk = %d", who, (long long)a.rows,
                (long long)a.vocab, (long long)a.row_stride, a.topk);
  if (!(a.temperature > 0.f) || !std::isfinite(a.temperature) || !std::isfinite(kLog2e / a.temperature))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: temperature = %g", who, (double)a.temperature);
  if (!std::isfinite(a.soft_weight) || !std::isfinite(a.hard_weight))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: soft_weight = %g, hard_weight = %g", who, (double)a.soft_weight,
                (double)a.hard_weight);
  return RAFHIP_OK;
}

int check_pointers(const char* who, const rafhip_topk_distill_args& a) {
  if ((a.vocab > 0 && !a.logits) || (a.topk > 0 && (!a.topk_indices || !a.topk_logits)))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: null tensor", who);
  if (!is_aligned(a.logits, element_bytes(a.logits_dtype)) || !is_aligned(a.topk_logits, element_bytes(a.topk_dtype)) ||
      !is_aligned(a.topk_indices, a.index_bits / 8) || !is_aligned(a.labels, a.index_bits / 8))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  return RAFHIP_OK;
}

int check_workspace(const char* who, int64_t need, const void* workspace, int64_t bytes) {
  if (need > 0 && (!workspace || bytes < need))
    return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p of %lld bytes, need %lld", who, workspace, (long long)bytes,
                (long long)need);
  if (need > 0 && !is_aligned(workspace, 16))
    return fail(RAFHIP_ERR_WORKSPACE, "%s: workspace %p is not 16-byte aligned", who, workspace);
  return RAFHIP_OK;
}

int check_gradient(const char* who, const rafhip_topk_distill_args& a, const float* dloss, int64_t dloss_count,
                   const void* dlogits, int64_t out_width) {
  if (dloss_count != a.rows && dloss_count != 1)
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: dloss has %lld values for %lld rows", who, (long long)dloss_count,
                (long long)a.rows);
  if (out_width < a.vocab) return fail(RAFHIP_ERR_INVALID_ARG, "%s: out_width = %lld < vocab", who, (long long)out_width);
  if (out_width >= (1LL << 28)) return fail(RAFHIP_ERR_UNSUPPORTED, "%s: out_width = %lld", who, (long long)out_width);
  if (a.rows > 0 && (!dloss || (out_width > 0 && !dlogits))) return fail(RAFHIP_ERR_INVALID_ARG, "%s: null tensor", who);
  if (!is_aligned(dloss, 4) || !is_aligned(dlogits, element_bytes(a.logits_dtype)))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  return RAFHIP_OK;
}

// Outputs against the inputs of every call, the gradient's own (none: NULL) and each other.
template <size_t kOuts>
int check_extents(const char* who, const rafhip_topk_distill_args& a, const Extent (&outs)[kOuts], const float* dloss = nullptr,
                  int64_t dloss_count = 0, const float* stats = nullptr) {
  const int64_t entries = a.rows * a.topk, index = a.index_bits / 8;
  const Extent ins[] = {
      {"logits", a.logits, a.vocab > 0 ? ((a.rows - 1) * a.row_stride + a.vocab) * element_bytes(a.logits_dtype) : 0},
      {"topk_indices", a.topk_indices, entries * index},
      {"topk_logits", a.topk_logits, entries * element_bytes(a.topk_dtype)},
      {"labels", a.labels, a.rows * index},
      {"dloss", dloss, dloss_count * 4},
      {"stats", stats, a.rows * 12}};
  return check_apart(who, outs, ins);
}

// A term that cannot matter is dropped here, so that the kernels neither read for it nor sum for it.
Task task_of(const rafhip_topk_distill_args& a, int* mode, float* c0) {
  Task t;
  t.logits = a.logits;
  t.indices = a.topk_indices;
  t.teacher = a.topk_logits;
  t.labels = a.hard_weight != 0.f ? a.labels : nullptr;
  t.rows = a.rows;
  t.row_stride = a.row_stride;
  t.vocab = (int)a.vocab;
  t.topk = a.soft_weight != 0.f ? a.topk : 0;
  t.teacher_dtype = a.topk_dtype;
  t.index_bits = a.index_bits;
  t.temperature = a.temperature;
  t.soft = a.soft_weight;
  t.hard = a.hard_weight;
  t.c_soft = (float)(1.44269504088896340736 / (double)a.temperature);
  const bool soft = t.topk > 0, hard = t.labels != nullptr;
  *mode = !soft || !hard || a.temperature == 1.f ? kOne
          : a.temperature == 2.f                    ? kSquare
          : a.temperature == 4.f                    ? kFourth
                                                    : kBoth;
  *c0 = soft ? t.c_soft : kLog2e;
  return t;
}

template <typename F>
void with_sums(int mode, F&& f) {
  if (mode == kOne)
    f(std::integral_constant<int, kOne>{});
  else if (mode == kBoth)
    f(std::integral_constant<int, kBoth>{});
  else if (mode == kSquare)
    f(std::integral_constant<int, kSquare>{});
  else
    f(std::integral_constant<int, kFourth>{});
}

constexpr int64_t kMaxGridY = 65535;
// Workgroups of `block` threads in a launch's first dimension.
int64_t max_grid_x(int block) { return kMaxGridBlocks * 256 / block; }

// Rows beyond the `most` that a launch's dimension holds go into further launches.
template <typename F>
void for_row_blocks(const Task& t, size_t element, int64_t most, F&& f) {
  for (int64_t r0 = 0; r0 < t.rows; r0 += most) {
    Task part = t;
    part.rows = t.rows - r0 < most ? t.rows - r0 : most;
    part.logits = static_cast<const char*>(t.logits) + (size_t)r0 * (size_t)t.row_stride * element;
    const size_t index = (size_t)t.index_bits / 8, teacher = t.teacher_dtype == RAFHIP_F32 ? 4 : 2;
    part.indices = static_cast<const char*>(t.indices) + (size_t)r0 * (size_t)t.topk * index;
    part.teacher = static_cast<const char*>(t.teacher) + (size_t)r0 * (size_t)t.topk * teacher;
    if (t.labels) part.labels = static_cast<const char*>(t.labels) + (size_t)r0 * index;
    f(part, r0);
  }
}

}  // namespace
}  // namespace rafhip

extern "C" int64_t rafhip_topk_distill_workspace_bytes(const rafhip_topk_distill_args* args) {
  using namespace rafhip;
  clear_error();
  if (check_args("rafhip_topk_distill_workspace_bytes", args) != RAFHIP_OK) return -1;
  const rafhip_topk_distill_args& a = *args;
  if (a.rows == 0 || a.vocab == 0) return 0;
  if (!loss_is_split(a.rows, a.vocab) && step_block(a.rows, a.vocab, a.logits_dtype) > 0) return 0;
  return parts_bytes(a.rows, a.vocab);
}

extern "C" int rafhip_topk_distill(const rafhip_topk_distill_args* args, float* loss, float* stats, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace rafhip;
  clear_error();
  const char* who = "rafhip_topk_distill";
  if (int st = check_args(who, args)) return st;
  const rafhip_topk_distill_args& a = *args;
  if (a.rows == 0) return RAFHIP_OK;
  if (int st = check_pointers(who, a)) return st;
  if (!loss) return fail(RAFHIP_ERR_INVALID_ARG, "%s: loss is NULL", who);
  if (!is_aligned(loss, 4) || !is_aligned(stats, 4))
    return fail(RAFHIP_ERR_INVALID_ARG, "%s: a tensor is not element-aligned", who);
  const bool split = loss_is_split(a.rows, a.vocab);
  const int64_t need = split ? parts_bytes(a.rows, a.vocab) : 0;
  if (int st = check_workspace(who, need, workspace, workspace_bytes)) return st;
  const Extent outs[] = {{"loss", loss, a.rows * 4}, {"stats", stats, a.rows * 12}, {"workspace", workspace, need}};
  if (int st = check_extents(who, a, outs)) return st;
  int sums;
  float c0;
  const Task t = task_of(a, &sums, &c0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_element(a.logits_dtype, [&](auto e) {
    with_sums(sums, [&](auto mode) {
      using T = decltype(e);
      constexpr int kSums = decltype(mode)::value;
      if (!split) {
        const int block = loss_block(a.rows, a.vocab);
        auto launch = [&](auto kernel) {
          for_row_blocks(t, sizeof(T), max_grid_x(block), [&](const Task& part, int64_t r0) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)part.rows), dim3((unsigned)block), 0, s, part, c0, loss + r0,
                               stats ? stats + r0 * 3 : nullptr);
          });
        };
        if (a.vocab > (int64_t)block * kMaxChain)
          launch(row_loss<T, kSums, true>);
        else
          launch(row_loss<T, kSums, false>);
        return;
      }
      float* parts = static_cast<float*>(workspace);
      const int per = columns_per_split(a.rows, a.vocab, kPartColumns), splits = (int)ceil_div(a.vocab, per);
      hipLaunchKernelGGL((row_part<T, kSums>), dim3((unsigned)splits, (unsigned)a.rows), dim3(kPartBlock), 0, s, t, c0,
                         per, parts);
      hipLaunchKernelGGL((join_loss<T, kSums>), dim3((unsigned)a.rows), dim3(kLanes), 0, s, t, c0, parts, splits, loss, stats);
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}

extern "C" int rafhip_topk_distill_dx(const rafhip_topk_distill_args* args, const float* dloss, int64_t dloss_count,
                                      const float* stats, void* dlogits, int64_t out_width, void* stream) {
  using namespace rafhip;
  clear_error();
  const char* who = "rafhip_topk_distill_dx";
  if (int st = check_args(who, args)) return st;
  const rafhip_topk_distill_args& a = *args;
  if (int st = check_gradient(who, a, dloss, dloss_count, dlogits, out_width)) return st;
  if (a.rows == 0 || out_width == 0) return RAFHIP_OK;
  if (int st = check_pointers(who, a)) return st;
  if (!stats || !is_aligned(stats, 4)) return fail(RAFHIP_ERR_INVALID_ARG, "%s: stats %p", who, (const void*)stats);
  const Extent outs[] = {{"dlogits", dlogits, a.rows * out_width * element_bytes(a.logits_dtype)}};
  if (int st = check_extents(who, a, outs, dloss, dloss_count, stats)) return st;
  int sums;
  float c0;
  const Task t = task_of(a, &sums, &c0);
  const int per = columns_per_split(a.rows, a.vocab, kGradColumns);
  const unsigned splits = (unsigned)(a.vocab > 0 ? ceil_div(a.vocab, per) : 1);
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_element(a.logits_dtype, [&](auto e) {
    with_sums(sums, [&](auto mode) {
      using T = decltype(e);
      constexpr int kSums = decltype(mode)::value;
      for_row_blocks(t, sizeof(T), kMaxGridY, [&](const Task& part, int64_t r0) {
        const int step = dloss_count == 1 ? 0 : 1;
        hipLaunchKernelGGL((row_grad<T, kSums>), dim3(splits, (unsigned)part.rows), dim3(kGradBlock),
                           picks_bytes(t.topk), s, part, c0, per, dloss + r0 * step, step, stats + r0 * 3,
                           (const float*)nullptr, 0, (float*)nullptr, static_cast<T*>(dlogits) + r0 * out_width, out_width,
                           picks_log2_slots(t.topk));
      });
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}

extern "C" int rafhip_topk_distill_step(const rafhip_topk_distill_args* args, const float* dloss, int64_t dloss_count,
                                        float* loss, void* dlogits, int64_t out_width, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  using namespace rafhip;
  clear_error();
  const char* who = "rafhip_topk_distill_step";
  if (int st = check_args(who, args)) return st;
  const rafhip_topk_distill_args& a = *args;
  if (int st = check_gradient(who, a, dloss, dloss_count, dlogits, out_width)) return st;
  if (a.rows == 0) return RAFHIP_OK;
  if (int st = check_pointers(who, a)) return st;
  if (!loss || !is_aligned(loss, 4)) return fail(RAFHIP_ERR_INVALID_ARG, "%s: loss %p", who, (const void*)loss);
  const int block = step_block(a.rows, a.vocab, a.logits_dtype);
  const int64_t need = block > 0 ? 0 : parts_bytes(a.rows, a.vocab);
  if (int st = check_workspace(who, need, workspace, workspace_bytes)) return st;
  const Extent outs[] = {{"loss", loss, a.rows * 4},
                         {"dlogits", dlogits, a.rows * out_width * element_bytes(a.logits_dtype)},
                         {"workspace", workspace, need}};
  if (int st = check_extents(who, a, outs, dloss, dloss_count)) return st;
  int sums;
  float c0;
  const Task t = task_of(a, &sums, &c0);
  const int step = dloss_count == 1 ? 0 : 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_element(a.logits_dtype, [&](auto e) {
    with_sums(sums, [&](auto mode) {
      using T = decltype(e);
      constexpr int kSums = decltype(mode)::value;
      if (block > 0) {
        with_step_kernel<T, kSums>((int)ceil_div(a.vocab / kWide, block), [&](auto kernel) {
          for_row_blocks(t, sizeof(T), max_grid_x(block), [&](const Task& part, int64_t r0) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)part.rows), dim3((unsigned)block), picks_bytes(t.topk), s, part, c0,
                               dloss + r0 * step, step, loss + r0, static_cast<T*>(dlogits) + r0 * out_width, out_width,
                               picks_log2_slots(t.topk));
          });
        });
        return;
      }
      const int per = columns_per_split(a.rows, a.vocab, kPartColumns), splits = (int)ceil_div(a.vocab, per);
      const int per_grad = columns_per_split(a.rows, a.vocab, kGradColumns);
      for_row_blocks(t, sizeof(T), kMaxGridY, [&](const Task& part, int64_t r0) {
        float* parts = static_cast<float*>(workspace) + r0 * splits * 4;
        hipLaunchKernelGGL((row_part<T, kSums>), dim3((unsigned)splits, (unsigned)part.rows), dim3(kPartBlock), 0, s, part, c0,
                           per, parts);
        hipLaunchKernelGGL((row_grad<T, kSums>), dim3((unsigned)ceil_div(a.vocab, per_grad) + 1, (unsigned)part.rows),
                           dim3(kGradBlock), picks_bytes(t.topk), s, part, c0, per_grad, dloss + r0 * step, step,
                           (const float*)nullptr, (const float*)parts, splits, loss + r0,
                           static_cast<T*>(dlogits) + r0 * out_width, out_width, picks_log2_slots(t.topk));
      });
    });
  });
  RAFHIP_HIP_TRY(hipGetLastError());
  return RAFHIP_OK;
}
