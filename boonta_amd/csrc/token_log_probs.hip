// Log probabilities of given tokens, entropies and top alternatives of rows of
// logits, and their vector-Jacobian product.
//
// Per row x of V logits, x_j = -inf where the mask does not allow j, temperature T:
//   w_j = (x_j - max x) / T, S = sum e^w, log p_j = w_j - ln S
//   log_prob = log p_token, entropy = ln S - sum e^w w / S
// (both sums of one sign, so neither cancels).  One pass: a thread keeps the
// maximum so far with S and sum e^w w relative to it, and rescales them when it
// grows.  A row that allows nothing has p = 0 and entropy 0.
// Backward: dx_j = (g (1_{j = token} - p_j) - h p_j (log p_j + entropy)) / T.
//
// The `top` largest x, equal ones by index.  A row held by a wave's lanes gives them one
// after the other.  Of a wider row a thread also keeps its best unit of 8 columns, by
// its largest value, then the lowest index.  The units of the `top` best threads hold
// the `top` best values: every one of those threads has a value that is better than
// all of any other thread.  So only their units are read again, those worse than the
// last of them left out, and ranked.
//
// What bounds it: HBM where rows are wide (8192 rows of 50001 bf16 logits 151 us, 5.4
// TB/s, backward 342, 4.8 TB/s), the vector work where they are short, a dozen
// instructions a column of a lane, there or not, and a hundred a row (262144 rows of
// 43 float32 logits with a mask 16 us, 3.8 TB/s, backward 21, 5.1 TB/s).  32 rows of
// 131072 with 8 alternatives take 12 us in 16 parts and 4 to join them, half of it the
// search.
#include "row_io.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace ppo;

enum TokenDtype { TOKEN_F32 = 0, TOKEN_BF16 = 1 };

constexpr int THREADS = 256, WAVES = THREADS / 64;
// With alternatives, rows of up to NARROW logits are a wave's lanes of up to four units (50M
// bf16 logits in rows of 2000, 8 alternatives 93 us, a workgroup a row 144; 20
// alternatives 195 for 212); where rows are few and alternatives more than FEW_TOP, of
// up to two (16 rows of 2000, 1 alternative 4.4 us for 7.1, 8 9.4 for 8.3).
// Without alternatives rows of up to SIDE are so, several a wave, and wider ones a wave
// each (400M bf16 logits in rows of 1030 241 us, a workgroup a row 680; of 2000 172 for
// 276, of 8000 150 for 159, but of 20000 151 for 139): up to WAVE_VOCAB, or where rows are
// few, and a row's time counts, up to FEW_VOCAB (1024 rows of 8000 8.8 us for 7.2 a
// workgroup a row, 4096 16.3 for 17.5; 64 of 2000 3.5 for 3.5).
constexpr int NARROW = 64 * UNIT * 4, SIDE = 32 * UNIT, FEW_TOP = 4;
constexpr int WAVE_VOCAB = 8192, FEW_VOCAB = 2048, WAVE_ROWS = 2048;
constexpr int WAVE_UNITS = 2;           // of a lane at a time (3 and 4 are level)
// Backward: widest row, in units, whose workgroup takes them one after the other, a few
// rows' together (400M bf16 logits, both passes: rows of 1030 970 us for 1780 a row a
// workgroup, of 4100 545 for 655, of 8000 440 for 460, but of 12000 462 for 449).
constexpr int FLAT_UNITS = 1024;
constexpr int MAX_TOP = 32;
constexpr int SEGMENT = 65536;          // most columns of a workgroup's part of a row
constexpr int MAX_SEGMENTS = 256;
constexpr int MAX_VOCAB = SEGMENT * MAX_SEGMENTS;
constexpr int BLOCKS = 16384;           // most workgroups of a launch over a wave's rows
constexpr int AHEAD = 4, BWD_AHEAD = 8; // units of a wide row that a thread has in flight
constexpr float LOWEST = -3.4028234663852886e38f, INF = __builtin_huge_valf();
constexpr float FAR = -1e30f;           // exponents below: 2^FAR = 0, and 0 FAR is a number
constexpr float LN2 = 0.6931471805599453f;

struct TokenArgs {
  const void* logits;
  const uint8_t* mask;      // or null
  const void* tokens;       // int32 or int64 [rows]
  float* log_prob;          // forward, [rows]
  float* entropy;
  float* stats;             // [rows, 2]: max, log2 S (forward: or null)
  float* top_log_probs;     // [rows, top]
  void* top_tokens;
  float* partials;          // rows in segments
  const float* dlog_prob;   // backward, each or null (zeros)
  const float* dentropy;
  void* dlogits;
  RowStride logits_s, mask_s, dlog_prob_s, dentropy_s;
  Divisor steps, units;     // units: of a row
  uint32_t rows;
  int V, top, lanes_log2, segments, segment_units, row_block;
  float c, inverse_t;       // log2(e) / T, 1 / T
  bool wide_tokens;
};

__device__ __forceinline__ int64_t token_of(const TokenArgs& p, uint32_t row) {
  return p.wide_tokens ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int32_t*>(p.tokens)[row];
}

// The mask's bytes of a unit at column col, 0 outside the row.
__device__ __forceinline__ uint64_t read_mask(const uint8_t* mask, int col, int V) {
  uint64_t allowed = 0;
  if (col >= 0 && col + UNIT <= V) {
    __builtin_memcpy(&allowed, mask + col, 8);
  } else {
#pragma unroll
    for (int j = 0; j < UNIT; ++j)
      if (col + j >= 0 && col + j < V) allowed |= (uint64_t)mask[col + j] << (8 * j);
  }
  return allowed;
}
// The 8 values of a unit, -inf where masked.
template <bool MASK, typename T>
__device__ __forceinline__ void unit_values(const Unit8<T>& raw, uint64_t allowed, float (&v)[UNIT]) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    v[j] = value(raw, j);
    if constexpr (MASK) v[j] = (allowed >> (8 * j)) & 0xff ? v[j] : -INF;
  }
}
// Those of any unit, -inf outside the row too.
template <bool MASK, typename T>
__device__ __forceinline__ void read_unit(const T* x, const uint8_t* mask, int col, int V, float (&v)[UNIT]) {
  Unit8<T> raw;
  if (col >= 0) load_unit(x + col, V - col, raw);
  else load_between(x + col, -col, V - col, raw);
  unit_values<MASK>(raw, MASK ? read_mask(mask, col, V) : 0, v);
#pragma unroll
  for (int j = 0; j < UNIT; ++j) v[j] = col + j >= 0 && col + j < V ? v[j] : -INF;
}
// Columns before a wide row's start from which its units are counted, so that
// they begin on a cache line (units that straddle 4-byte words load at 5.0 TB/s for
// 6.0; a wave's stores are whole lines).
template <typename T> __device__ __forceinline__ int skew_of(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 127) / sizeof(T));
}
constexpr int MAX_SKEW = 63;
__device__ __forceinline__ float max8(const float (&v)[UNIT]) {
  return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}

// Maximum, sum of 2^w and sum of 2^w w, w = (x - maximum) c.
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums no_sums() { return Sums{LOWEST, 0.f, 0.f}; }
__device__ __forceinline__ float exponent(float x, float m, float c) { return (x - m) * c; }
// (an infinite x or a NaN makes s NaN, and so the row's results)
__device__ __forceinline__ Sums rescaled(const Sums& a, float m, float c) {
  const float d = exponent(a.m, m, c), f = __builtin_amdgcn_exp2f(d);
  return Sums{m, a.s * f, f * __fmaf_rn(fmaxf(d, FAR), a.s, a.t)};
}
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = rescaled(a, m, c), y = rescaled(b, m, c);
  return Sums{m, x.s + y.s, x.t + y.t};
}
// The unit's own sums first: a thread's are of an eighth of the terms, which a far larger one would each round.
__device__ __forceinline__ void add_values(Sums& a, const float (&v)[UNIT], float c) {   // none above a.m
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    const float w = exponent(v[j], a.m, c), e = __builtin_amdgcn_exp2f(w);
    s += e;
    t = __fmaf_rn(e, fmaxf(w, FAR), t);
  }
  a.s += s;
  a.t += t;
}
__device__ __forceinline__ void add_unit(Sums& a, const float (&v)[UNIT], float most, float c) {
  a = rescaled(a, fmaxf(a.m, most), c);
  add_values(a, v, c);
}
// Over 2^log2 neighbouring lanes (all active): one change of the maximum, not one a
// stage (64 rows of 50000 bf16 logits 8.5 -> 7.9 us).
__device__ __forceinline__ Sums lanes_joined(Sums a, int log2, float c) {
  a = rescaled(a, lanes_max(a.m, log2), c);
  a.s = lanes_sum(a.s, log2);
  a.t = lanes_sum(a.t, log2);
  return a;
}

// log p of a logit, l = log2 S: from halves, whose difference every pair of float32 numbers has (-3e38 less 3e38, or
// the type's lowest value as a mask), times 1 / T at once.
__device__ __forceinline__ float log_p(const TokenArgs& p, float x, float m, float l) {
  return __fmaf_rn(0.5f * x - 0.5f * m, 2.f * p.inverse_t, -LN2 * l);
}

// The row's token: its logit where it is one that is allowed.
struct Given {
  bool token;
  float logit;   // -inf: not allowed
};
template <typename T>
__device__ __forceinline__ Given given_of(const TokenArgs& p, uint32_t row, const T* x, const uint8_t* mask) {
  const int64_t token = token_of(p, row);
  Given g{token >= 0 && token < p.V, -INF};
  if (g.token && !(mask && !mask[token])) {
    if constexpr (sizeof(T) == 2) g.logit = __uint_as_float((uint32_t)x[token] << 16);
    else g.logit = x[token];
  }
  return g;
}
// A row's results from its sums, by one thread.
__device__ __forceinline__ void finish_row(const TokenArgs& p, uint32_t row, const Sums& a, const Given& g) {
  const bool none = a.s == 0.f;
  const float l = none ? INF : __builtin_amdgcn_logf(a.s);   // log2
  p.entropy[row] = none ? 0.f : LN2 * (l - a.t * __builtin_amdgcn_rcpf(a.s));   // (S from 1 to 2^24)
  p.log_prob[row] = !g.token ? 0.f : g.logit == -INF ? -INF : log_p(p, g.logit, a.m, l);
  if (p.stats) {
    p.stats[2 * (int64_t)row] = none ? 0.f : a.m;
    p.stats[2 * (int64_t)row + 1] = l;
  }
}

// ---- top alternatives
// A key orders values, equal ones by the lower index; 0: no value (masked, or NaN).
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t ordered = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x > -INF ? (uint64_t)ordered << 32 | (uint32_t)~index : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ void write_top(const TokenArgs& p, uint32_t row, int place, float x, int token, float m, float l) {
  const int64_t at = (int64_t)row * p.top + place;
  p.top_log_probs[at] = token < 0 ? -INF : log_p(p, x, m, l);
  if (p.wide_tokens) static_cast<int64_t*>(p.top_tokens)[at] = token;
  else static_cast<int32_t*>(p.top_tokens)[at] = token;
}
__device__ __forceinline__ void write_top(const TokenArgs& p, uint32_t row, int place, uint64_t key, float m, float l) {
  write_top(p, row, place, value_of(key), key ? (int32_t)index_of(key) : -1, m, l);
}

// ---- rows of lanes of a wave
// Unit u of a row: the row's last 8 columns where it would pass the end,
// the first `skip` of them in the unit before too (all 8 or more past the end).
struct Span {
  int col, skip;
};
__device__ __forceinline__ Span span_of(int u, int V) {
  const int col = max(0, min(u * UNIT, V - UNIT));
  return Span{col, u * UNIT - col};
}
template <bool MASK, typename T>
__device__ __forceinline__ void read_span(const T* x, const uint8_t* mask, const Span& at, int V, float (&v)[UNIT]) {
  if (V >= UNIT) {
    Unit8<T> raw;
    __builtin_memcpy(raw.w, x + at.col, sizeof(raw.w));
    uint64_t allowed = 0;
    if constexpr (MASK) __builtin_memcpy(&allowed, mask + at.col, 8);
    unit_values<MASK>(raw, allowed, v);
  } else {
    read_unit<MASK>(x, mask, 0, V, v);
  }
}

// U: units of a lane (those of a row's lanes side by side).  LOG2: of the lanes, -1: as
// given (known, 100M bf16 logits in rows of 43 122 -> 89 us).
template <typename T, bool TOP, bool MASK, int U, int LOG2>
__global__ void __launch_bounds__(THREADS) token_narrow_kernel(TokenArgs p) {
  const int log2 = LOG2 < 0 ? p.lanes_log2 : LOG2, L = 1 << log2, lane = threadIdx.x & (L - 1);
  Span at[U];
#pragma unroll
  for (int k = 0; k < U; ++k) at[k] = span_of(lane + k * L, p.V);
  const uint32_t step = (gridDim.x * THREADS) >> log2;
  for (uint32_t row0 = (blockIdx.x * THREADS + threadIdx.x) >> log2; __any(row0 < p.rows); row0 += step) {
    const bool live = row0 < p.rows;
    const uint32_t row = live ? row0 : p.rows - 1;
    const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
    const uint8_t* mask = MASK ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr;
    Given given{};
    if (lane == 0) given = given_of(p, row, x, mask);
    float v[U][UNIT], most = -INF;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      read_span<MASK>(x, mask, at[k], p.V, v[k]);
#pragma unroll
      for (int j = 0; j < UNIT; ++j) v[k][j] = j >= at[k].skip ? v[k][j] : -INF;
      most = fmaxf(most, max8(v[k]));
    }
    Sums a{fmaxf(most, LOWEST), 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < U; ++k) add_values(a, v[k], p.c);
    a = lanes_joined(a, log2, p.c);
    if (live && lane == 0) finish_row(p, row, a, given);
    if constexpr (TOP) {
      const float l = __builtin_amdgcn_logf(a.s);
      // one after the other: the row's largest value, the lowest of its columns (as a
      // float: below 2^24), and out with it; lane n of the row's keeps the n-th, and
      // every L of them are written together
      float kept = -INF;
      int kept_col = -1;
      for (int n = 0; n < p.top; ++n) {
        most = max8(v[0]);
#pragma unroll
        for (int k = 1; k < U; ++k) most = fmaxf(most, max8(v[k]));
        most = lanes_max(most, log2);
        float at_most = -INF;   // less its column
#pragma unroll
        for (int k = U - 1; k >= 0; --k)
#pragma unroll
          for (int j = UNIT - 1; j >= 0; --j) at_most = v[k][j] == most ? -(float)(at[k].col + j) : at_most;
        at_most = lanes_max(at_most, log2);
        const int col = most > -INF ? (int)-at_most : -1;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int away = col - at[k].col;
#pragma unroll
          for (int j = 0; j < UNIT; ++j) v[k][j] = away == j ? -INF : v[k][j];
        }
        const int place = n & (L - 1);
        kept = lane == place ? most : kept;
        kept_col = lane == place ? col : kept_col;
        if (place == L - 1 || n == p.top - 1) {
          if (live && lane <= place) write_top(p, row, n - place + lane, kept, kept_col, a.m, l);
        }
      }
    }
  }
}

// A wave for each row, WAVE_UNITS of a lane at a time, as many as there are: an empty unit
// costs the vector work of a full one, which bounds rows of few (1030 logits 299 -> 241 us).
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) token_wave_kernel(TokenArgs p) {
  const int lane = threadIdx.x & 63, units = (int)p.units.d;
  for (uint32_t row = blockIdx.x * WAVES + (threadIdx.x >> 6); row < p.rows; row += gridDim.x * WAVES) {
    const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
    const uint8_t* mask = MASK ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr;
    Given given{};
    if (lane == 0) given = given_of(p, row, x, mask);
    Sums a = no_sums();
    for (int u0 = 0; u0 < units; u0 += 64 * WAVE_UNITS) {
      Unit8<T> raw[WAVE_UNITS];
      uint64_t allowed[WAVE_UNITS];
#pragma unroll
      for (int k = 0; k < WAVE_UNITS; ++k) {
        if (u0 + 64 * k >= units) continue;   // (of the whole wave)
        const Span at = span_of(u0 + 64 * k + lane, p.V);
        __builtin_memcpy(raw[k].w, x + at.col, sizeof(raw[k].w));
        if constexpr (MASK) __builtin_memcpy(&allowed[k], mask + at.col, 8);
      }
#pragma unroll
      for (int k = 0; k < WAVE_UNITS; ++k) {
        if (u0 + 64 * k >= units) continue;
        const Span at = span_of(u0 + 64 * k + lane, p.V);
        float v[UNIT];
        unit_values<MASK>(raw[k], MASK ? allowed[k] : 0, v);
#pragma unroll
        for (int j = 0; j < UNIT; ++j) v[j] = j >= at.skip ? v[j] : -INF;
        add_unit(a, v, max8(v), p.c);
      }
    }
    a = lanes_joined(a, 6, p.c);
    if (lane == 0) finish_row(p, row, a, given);
  }
}

// ---- wider rows: a workgroup for each row, or each segment of it
// What a segment leaves: its sums, then its best keys.
__device__ __forceinline__ int64_t partial_floats(int top) { return 4 + 2 * top; }

constexpr int MOST_UNITS = MAX_TOP * (SEGMENT / (UNIT * THREADS) + 1);   // of the best threads
struct TopSpace {
  uint64_t lists[WAVES * MAX_TOP];   // each wave's best keys, in order; 0: none
  uint64_t best[MAX_TOP];            // and those of all
  uint64_t candidates[MOST_UNITS];
  uint64_t values[MAX_TOP * UNIT];
  uint32_t units[MAX_TOP];
  int count;
};

// A key's rank: how many of n are better.
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* keys, int n) {
  int r = 0, i = 0;
  for (; i + 8 <= n; i += 8) {   // (reads of eight on their way at once)
    uint64_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = keys[i + j];
#pragma unroll
    for (int j = 0; j < 8; ++j) r += k[j] > key;
  }
  for (; i < n; ++i) r += keys[i] > key;
  return r;
}
// Among the keys of the wave.
__device__ __forceinline__ int rank_in_wave(uint64_t key) {
  int r = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), i) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)key, i);
    r += other > key;
  }
  return r;
}
// The best keys of lists, `top` of each in order (0: no more), in order; `n` lists of
// `pitch` keys.  Rooms of the workgroup's; ends with a barrier.
__device__ __forceinline__ void merge_lists(const uint64_t* lists, int n, int pitch, int top, uint64_t* best) {
  const int tid = threadIdx.x;
  if (tid < top) best[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n * top; i += THREADS) {
    const uint64_t key = lists[(i / top) * pitch + i % top];
    int r = 0;
    for (int w = 0; w < n; ++w) r += rank_of(key, lists + w * pitch, top);
    if (key && r < top) best[r] = key;
  }
  __syncthreads();
}

template <typename T, bool TOP, bool MASK>
__global__ void __launch_bounds__(THREADS) token_wide_kernel(TokenArgs p) {
  __shared__ Sums sums[WAVES];
  __shared__ typename std::conditional<TOP, TopSpace, int>::type space;
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
  const uint8_t* mask = MASK ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr;
  const int skew = skew_of(x), first = blockIdx.y * p.segment_units;
  const int end = min((p.V + skew + UNIT - 1) / UNIT, first + p.segment_units), whole = min(end, (p.V + skew) / UNIT);
  x -= skew;   // (columns in the units' count from here on; those before the row are not read)
  if constexpr (MASK) mask -= skew;
  Sums a = no_sums();
  float best = -INF;
  int best_unit = 0;
  auto read = [&](int u, float (&v)[UNIT]) __attribute__((always_inline)) {
    read_unit<MASK>(x + skew, mask + skew, u * UNIT - skew, p.V, v);
  };
  auto add = [&](const float (&v)[UNIT], int u) __attribute__((always_inline)) {
    const float most = max8(v);
    add_unit(a, v, most, p.c);
    if constexpr (TOP) {
      best_unit = most > best ? u : best_unit;
      best = most > best ? most : best;
    }
  };
  int u = first + tid;
  if (u * UNIT < skew && u < end) {   // the row's first columns
    float v[UNIT];
    read(u, v);
    add(v, u);
    u += THREADS;
  }
  for (; u + (AHEAD - 1) * THREADS < whole; u += AHEAD * THREADS) {
    Unit8<T> raw[AHEAD];
    uint64_t allowed[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      load_unit_once(x + (u + k * THREADS) * UNIT, raw[k]);
      if constexpr (MASK) __builtin_memcpy(&allowed[k], mask + (u + k * THREADS) * UNIT, 8);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      float v[UNIT];
      unit_values<MASK>(raw[k], MASK ? allowed[k] : 0, v);
      add(v, u + k * THREADS);
    }
  }
  for (; u < end; u += THREADS) {
    float v[UNIT];
    read(u, v);
    add(v, u);
  }
  a = lanes_joined(a, 6, p.c);
  if ((tid & 63) == 0) sums[tid >> 6] = a;
  if constexpr (TOP) {
    // the best threads of each wave, in order
    const uint64_t mine = key_of(best, (uint32_t)best_unit);
    uint64_t* list = space.lists + (tid >> 6) * MAX_TOP;
    if ((tid & 63) < MAX_TOP) list[tid & 63] = 0;
    const int rank = rank_in_wave(mine);
    if (mine && rank < p.top) list[rank] = mine;
    if (tid == 0) space.count = 0;
  }
  __syncthreads();
  a = sums[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) a = joined(a, sums[w], p.c);
  float* partial = p.partials + ((int64_t)row * p.segments + blockIdx.y) * partial_floats(p.top);
  if (tid == 0) {
    if (p.segments == 1) {
      finish_row(p, row, a, given_of(p, row, x + skew, MASK ? mask + skew : nullptr));
    } else {
      partial[0] = a.m;
      partial[1] = a.s;
      partial[2] = a.t;
    }
  }
  if constexpr (TOP) {
    merge_lists(space.lists, WAVES, MAX_TOP, p.top, space.best);
    // of the best threads' units those no worse than the last thread's best
    const uint64_t held = (tid & 63) < p.top ? space.best[tid & 63] : 0;
    const int threads = __popcll(__ballot(held != 0));
    const uint64_t least = threads < p.top ? 1 : space.best[p.top - 1];
    const int each = (end - first + THREADS - 1) / THREADS;
    for (int i = tid; i < threads * each; i += THREADS) {
      const int w = i / each;
      const int thread = ((int)index_of(space.best[w]) - first) % THREADS, u = first + thread + (i - w * each) * THREADS;
      if (u >= end) continue;
      float v[UNIT];
      read(u, v);
      const uint64_t key = key_of(max8(v), (uint32_t)u);
      if (key >= least) space.candidates[atomicAdd(&space.count, 1)] = key;
    }
    __syncthreads();
    // the best units among them, and of those the best values
    const int candidates = space.count, units = min(candidates, p.top);
    for (int i = tid; i < candidates; i += THREADS) {
      const uint64_t key = space.candidates[i];
      const int r = rank_of(key, space.candidates, candidates);
      if (r < p.top) space.units[r] = index_of(key);
    }
    if (tid < MAX_TOP) space.best[tid] = 0;
    __syncthreads();
    uint64_t value = 0;
    if (tid < units * UNIT) {
      float v[UNIT];
      const int u = (int)space.units[tid / UNIT];
      read(u, v);
      float one = -INF;
#pragma unroll
      for (int j = 0; j < UNIT; ++j) one = tid % UNIT == j ? v[j] : one;
      value = key_of(one, (uint32_t)(u * UNIT - skew + tid % UNIT));
      space.values[tid] = value;
    }
    __syncthreads();
    if (value) {
      const int r = rank_of(value, space.values, units * UNIT);
      if (r < p.top) space.best[r] = value;
    }
    __syncthreads();
    if (tid < p.top) {
      if (p.segments == 1) write_top(p, row, tid, space.best[tid], a.m, __builtin_amdgcn_logf(a.s));
      else __builtin_memcpy(partial + 4 + 2 * tid, &space.best[tid], 8);
    }
  }
}

// A row's segments joined: the sums by the first wave; of the segments whose best
// key is among the `top` best of all segments' the keys, and of those the best.
template <typename T> __global__ void __launch_bounds__(THREADS) token_join_kernel(TokenArgs p) {
  __shared__ uint64_t heads[MAX_SEGMENTS], lists[MAX_TOP * MAX_TOP], best[MAX_TOP];
  __shared__ Sums sums;
  __shared__ int from[MAX_TOP];
  const uint32_t row = blockIdx.x;
  const int tid = threadIdx.x, pitch = (int)partial_floats(p.top);
  const float* partial = p.partials + (int64_t)row * p.segments * pitch;
  if (tid < 64) {
    const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
    Given given{};
    if (tid == 0) given = given_of(p, row, x, p.mask ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr);
    Sums a = no_sums();
    for (int s = tid; s < p.segments; s += 64) {
      const float* q = partial + s * pitch;
      a = joined(a, Sums{q[0], q[1], q[2]}, p.c);
    }
    a = lanes_joined(a, 6, p.c);
    if (tid == 0) {
      sums = a;
      finish_row(p, row, a, given);
    }
  }
  if (p.top == 0) return;
  auto key_at = [&](int segment, int place) {
    uint64_t key;
    __builtin_memcpy(&key, partial + segment * pitch + 4 + 2 * place, 8);
    return key;
  };
  uint64_t mine = 0;
  if (tid < p.segments) heads[tid] = mine = key_at(tid, 0);
  if (tid < MAX_TOP) from[tid] = -1;
  __syncthreads();
  if (mine) {
    const int r = rank_of(mine, heads, p.segments);
    if (r < p.top) from[r] = tid;
  }
  __syncthreads();
  for (int i = tid; i < p.top * p.top; i += THREADS) {
    const int segment = from[i / p.top];
    lists[(i / p.top) * MAX_TOP + i % p.top] = segment < 0 ? 0 : key_at(segment, i % p.top);
  }
  __syncthreads();
  merge_lists(lists, p.top, MAX_TOP, p.top, best);
  if (tid < p.top) write_top(p, row, tid, best[tid], sums.m, __builtin_amdgcn_logf(sums.s));
}

// ---- backward: a workgroup takes `row_block` rows' units, or a segment of one row's
// What a row's gradients need: dx = -2^w (hl max(w, .) + gh) with w = (x - m) c - l,
// hl = h ln(2) / T, gh = (g + h entropy) / T; and g / T at the token.
struct RowGradient {
  float m, l, hl, gh, g;
  int token;   // -1: none
  bool bad;    // a logit or cotangent that is not finite: NaN, but where the mask allows nothing
};
constexpr float LEAST = -200.f;   // exponents below: 2^LEAST = 0
template <typename T> __device__ __forceinline__ RowGradient row_gradient(const TokenArgs& p, uint32_t row) {
  RowGradient r;
  r.m = p.stats[2 * (int64_t)row];
  r.l = p.stats[2 * (int64_t)row + 1];
  const int64_t token = token_of(p, row);
  // a token that is none, or not allowed, passes nothing (its log probability is -inf, which an allowed one's may be)
  bool given = token >= 0 && token < p.V;
  if (given && p.log_prob[row] == -INF) {
    const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
    given = given_of(p, row, x, p.mask ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr).logit > -INF;
  }
  r.token = given ? (int)token : -1;
  r.g = given && p.dlog_prob ? p.dlog_prob[row_offset(row, p.steps, p.dlog_prob_s)] * p.inverse_t : 0.f;
  const float h = p.dentropy ? p.dentropy[row_offset(row, p.steps, p.dentropy_s)] * p.inverse_t : 0.f;
  r.hl = h * LN2;
  r.gh = __fmaf_rn(h, p.entropy[row], r.g);
  r.bad = r.l != r.l || !(__fmaf_rn(fabsf(r.hl), -LEAST, fabsf(r.gh)) < INF);
  return r;
}
__device__ __forceinline__ void unit_gradient(const RowGradient& r, float c, int col, float (&v)[UNIT]) {
  float d[UNIT];
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    const float w = __fmaf_rn(v[j] - r.m, c, -r.l), e = __builtin_amdgcn_exp2f(w);
    d[j] = -e * __fmaf_rn(r.hl, fmaxf(w, LEAST), r.gh);
  }
  if (r.bad) {
    asm volatile("");   // (seldom: not selected from beside the others)
#pragma unroll
    for (int j = 0; j < UNIT; ++j) d[j] = v[j] == -INF ? 0.f : d[j];
  }
  const int at = r.token - col;
  if (at >= 0 && at < UNIT) {
    asm volatile("");
#pragma unroll
    for (int j = 0; j < UNIT; ++j) d[j] = j == at ? d[j] + r.g : d[j];   // (-0 stays: a unit that overlaps this one writes it)
  }
#pragma unroll
  for (int j = 0; j < UNIT; ++j) v[j] = d[j];
}

// Rows of up to FLAT_UNITS: several side by side, their scalars formed once in LDS.
constexpr int MAX_ROW_BLOCK = 256;
template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) token_bwd_kernel(TokenArgs p) {
  __shared__ RowGradient scalars[MAX_ROW_BLOCK];
  const uint32_t units = p.units.d, row0 = blockIdx.x * p.row_block;
  const uint32_t rows = min((uint32_t)p.row_block, p.rows - row0), count = rows * units;
  if (threadIdx.x < rows) scalars[threadIdx.x] = row_gradient<T>(p, row0 + threadIdx.x);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
    const uint32_t q = quotient(i, p.units), row = row0 + q;
    const Span at = span_of((int)(i - q * units), p.V);
    float v[UNIT];
    read_span<MASK>(static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s),
                    MASK ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr, at, p.V, v);
    unit_gradient(scalars[q], p.c, at.col, v);
    store_unit(static_cast<T*>(p.dlogits) + (int64_t)row * p.V + at.col, min(p.V, UNIT), v);
  }
}

template <typename T, bool MASK> __global__ void __launch_bounds__(THREADS) token_bwd_wide_kernel(TokenArgs p) {
  const uint32_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row_offset(row, p.steps, p.logits_s);
  const uint8_t* mask = MASK ? p.mask + row_offset(row, p.steps, p.mask_s) : nullptr;
  T* out = static_cast<T*>(p.dlogits) + (int64_t)row * p.V;
  const int skew = skew_of(out), first = blockIdx.y * p.segment_units;   // (as the logits where those are contiguous)
  const int end = min((p.V + skew + UNIT - 1) / UNIT, first + p.segment_units), whole = min(end, (p.V + skew) / UNIT);
  const RowGradient r = row_gradient<T>(p, row);
  auto one = [&](int u) __attribute__((always_inline)) {
    const int col = u * UNIT - skew;
    float v[UNIT];
    read_unit<MASK>(x, mask, col, p.V, v);
    unit_gradient(r, p.c, col, v);
    store_between(out + col, -col, p.V - col, v);
  };
  int u = first + threadIdx.x;
  if (u * UNIT < skew && u < end) {   // the row's first columns
    one(u);
    u += THREADS;
  }
  for (; u + (BWD_AHEAD - 1) * THREADS < whole; u += BWD_AHEAD * THREADS) {
    Unit8<T> raw[BWD_AHEAD];
    uint64_t allowed[BWD_AHEAD];
#pragma unroll
    for (int k = 0; k < BWD_AHEAD; ++k) {
      const int col = (u + k * THREADS) * UNIT - skew;
      load_unit_once(x + col, raw[k]);
      if constexpr (MASK) __builtin_memcpy(&allowed[k], mask + col, 8);
    }
#pragma unroll
    for (int k = 0; k < BWD_AHEAD; ++k) {
      const int col = (u + k * THREADS) * UNIT - skew;
      float v[UNIT];
      unit_values<MASK>(raw[k], MASK ? allowed[k] : 0, v);
      unit_gradient(r, p.c, col, v);
      store_unit(out + col, UNIT, v);
    }
  }
  for (; u < whole; u += THREADS) {
    const int col = u * UNIT - skew;
    float v[UNIT];
    read_unit<MASK>(x, mask, col, p.V, v);
    unit_gradient(r, p.c, col, v);
    store_unit(out + col, UNIT, v);
  }
  if (u < end) one(u);   // and its last
}

// ---- launches
int check(const char* what, int dtype, int batch, int steps, int vocab, float temperature) {
  if (dtype != TOKEN_F32 && dtype != TOKEN_BF16) return set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || vocab < 1 || vocab > MAX_VOCAB)
    return set_error(PPO_ERR_ARG, "%s: bad size (batch %d steps %d vocabulary %d of 1 .. %d)", what, batch, steps, vocab,
                     MAX_VOCAB);
  if ((int64_t)batch * steps > (1 << 24) - 1)
    return set_error(PPO_ERR_ARG, "%s: batch x steps above 2^24 - 1", what);
  if (!(temperature >= 1e-30f && temperature <= 1e30f))   // (its inverse is a float32 number)
    return set_error(PPO_ERR_ARG, "%s: temperature %g is not from 1e-30 to 1e30", what, (double)temperature);
  return PPO_OK;
}

// Parts of a wide row, where rows are few and long: about two for each CU, of at
// least 8192 columns (32 rows of 131072 bf16 logits, 8 alternatives: 15.7 us for
// 19.4 in one part; 32768 columns gain nothing, 1 row 11.5 for 12.6 us, and 5000
// lose the join's 2 to 4 us).  With alternatives no part is longer than SEGMENT.
int segments_of(int64_t rows, int vocab, int top) {
  if (vocab <= 32768 || rows == 0) return 1;
  const int64_t fill = std::min(ceil_div64(512, rows), ceil_div64(vocab, 8192));
  return (int)std::min<int64_t>(MAX_SEGMENTS, std::max(fill, top ? ceil_div64(vocab, SEGMENT) : 1));
}

TokenArgs common_args(const void* logits, const void* tokens, int wide_tokens, const uint8_t* mask,
                      const int64_t* strides, float temperature, int batch, int steps, int vocab) {
  TokenArgs a{};
  a.logits = logits;
  a.mask = mask;
  a.tokens = tokens;
  a.logits_s = RowStride{strides[0], strides[1]};
  a.mask_s = RowStride{strides[2], strides[3]};
  a.steps = divisor((uint32_t)steps);
  a.units = divisor((uint32_t)ceil_div(vocab, UNIT));
  a.rows = (uint32_t)((int64_t)batch * steps);
  a.V = vocab;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.inverse_t = (float)(1.0 / (double)temperature);
  a.wide_tokens = wide_tokens != 0;
  return a;
}

template <typename T, bool MASK> void launch_fwd(hipStream_t st, TokenArgs& a) {
  if (!a.top && a.V > SIDE && a.V <= (a.rows >= WAVE_ROWS ? WAVE_VOCAB : FEW_VOCAB)) {
    const dim3 blocks((unsigned)std::min<int64_t>(BLOCKS, ceil_div64(a.rows, WAVES)));
    hipLaunchKernelGGL((token_wave_kernel<T, MASK>), blocks, dim3(THREADS), 0, st, a);
    return;
  }
  if (a.V <= (a.rows >= WAVE_ROWS || a.top <= FEW_TOP ? NARROW : NARROW / 2)) {
    while (a.lanes_log2 < 6 && (UNIT << a.lanes_log2) < a.V) ++a.lanes_log2;
    const dim3 blocks((unsigned)std::min<int64_t>(BLOCKS, ceil_div64((int64_t)a.rows << a.lanes_log2, THREADS)));
    const auto lanes = [&](auto log2) {
      hipLaunchKernelGGL((token_narrow_kernel<T, false, MASK, 1, decltype(log2)::value>), blocks, dim3(THREADS), 0, st, a);
    };
    if (a.top && a.V > 128 * UNIT) hipLaunchKernelGGL((token_narrow_kernel<T, true, MASK, 4, 6>), blocks, dim3(THREADS), 0, st, a);
    else if (a.top && a.V > 64 * UNIT) hipLaunchKernelGGL((token_narrow_kernel<T, true, MASK, 2, 6>), blocks, dim3(THREADS), 0, st, a);
    else if (a.top) hipLaunchKernelGGL((token_narrow_kernel<T, true, MASK, 1, -1>), blocks, dim3(THREADS), 0, st, a);
    else if (a.lanes_log2 == 0) lanes(std::integral_constant<int, 0>{});
    else if (a.lanes_log2 == 1) lanes(std::integral_constant<int, 1>{});
    else if (a.lanes_log2 == 2) lanes(std::integral_constant<int, 2>{});
    else if (a.lanes_log2 == 3) lanes(std::integral_constant<int, 3>{});
    else if (a.lanes_log2 == 4) lanes(std::integral_constant<int, 4>{});
    else lanes(std::integral_constant<int, 5>{});
    return;
  }
  const dim3 grid(a.rows, a.segments);
  if (a.top) hipLaunchKernelGGL((token_wide_kernel<T, true, MASK>), grid, dim3(THREADS), 0, st, a);
  else hipLaunchKernelGGL((token_wide_kernel<T, false, MASK>), grid, dim3(THREADS), 0, st, a);
  if (a.segments > 1) hipLaunchKernelGGL((token_join_kernel<T>), dim3(a.rows), dim3(a.top ? THREADS : 64), 0, st, a);
}

template <typename T, bool MASK> void launch_bwd(hipStream_t st, TokenArgs& a) {
  const int units = (int)a.units.d;
  a.row_block = std::min(MAX_ROW_BLOCK, std::max(1, 4 * THREADS / units));
  const int most = ceil_div(a.V + MAX_SKEW, UNIT);
  const int segments = ceil_div(most, 8 * THREADS);
  a.segment_units = ceil_div(most, segments);
  if (units <= FLAT_UNITS)
    hipLaunchKernelGGL((token_bwd_kernel<T, MASK>), dim3((unsigned)ceil_div64(a.rows, a.row_block)), dim3(THREADS), 0, st, a);
  else
    hipLaunchKernelGGL((token_bwd_wide_kernel<T, MASK>), dim3(a.rows, (unsigned)segments), dim3(THREADS), 0, st,
                       a);
}

}  // namespace

PPO_EXPORT int ppo_token_log_probs_max_top(void) { return MAX_TOP; }
PPO_EXPORT int ppo_token_log_probs_max_vocab(void) { return MAX_VOCAB; }

PPO_EXPORT size_t ppo_token_log_probs_workspace(int batch, int steps, int vocab, int top) {
  if (batch <= 0 || steps <= 0 || vocab <= NARROW || vocab > MAX_VOCAB || top < 0 || top > MAX_TOP) return 0;
  const int64_t rows = (int64_t)batch * steps;
  const int s = segments_of(rows, vocab, top);
  return s > 1 ? sizeof(float) * (size_t)(4 + 2 * top) * (size_t)rows * s : 0;
}

PPO_EXPORT int ppo_token_log_probs_fwd(void* stream, int dtype, const void* logits, const void* tokens,
                                       int wide_tokens, const uint8_t* mask, const int64_t* strides,
                                       float temperature, int top, float* log_prob, float* entropy, float* stats,
                                       float* top_log_probs, void* top_tokens, void* workspace,
                                       size_t workspace_bytes, int batch, int steps, int vocab) {
  const char* what = "ppo_token_log_probs_fwd";
  if (int rc = check(what, dtype, batch, steps, vocab, temperature)) return rc;
  if (top < 0 || top > MAX_TOP) return set_error(PPO_ERR_ARG, "%s: %d alternatives of 0 .. %d", what, top, MAX_TOP);
  if ((int64_t)batch * steps == 0) return PPO_OK;
  if (!logits || !tokens || !strides || !log_prob || !entropy || (top > 0 && (!top_log_probs || !top_tokens)))
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  const size_t need = ppo_token_log_probs_workspace(batch, steps, vocab, top);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  TokenArgs a = common_args(logits, tokens, wide_tokens, mask, strides, temperature, batch, steps, vocab);
  a.log_prob = log_prob;
  a.entropy = entropy;
  a.stats = stats;
  a.top = top;
  a.top_log_probs = top_log_probs;
  a.top_tokens = top_tokens;
  a.partials = static_cast<float*>(workspace);
  a.segments = segments_of(a.rows, vocab, top);
  a.segment_units = ceil_div(ceil_div(vocab + MAX_SKEW, UNIT), a.segments);
  if (dtype == TOKEN_F32) mask ? launch_fwd<float, true>(as_stream(stream), a) : launch_fwd<float, false>(as_stream(stream), a);
  else mask ? launch_fwd<uint16_t, true>(as_stream(stream), a) : launch_fwd<uint16_t, false>(as_stream(stream), a);
  return check_launch(what);
}

PPO_EXPORT int ppo_token_log_probs_bwd(void* stream, int dtype, const void* logits, const void* tokens,
                                       int wide_tokens, const uint8_t* mask, const int64_t* strides,
                                       float temperature, const float* log_prob, const float* entropy,
                                       const float* stats, const float* dlog_prob, const float* dentropy,
                                       void* dlogits, int batch, int steps, int vocab) {
  const char* what = "ppo_token_log_probs_bwd";
  if (int rc = check(what, dtype, batch, steps, vocab, temperature)) return rc;
  if ((int64_t)batch * steps == 0) return PPO_OK;
  if (!logits || !tokens || !strides || !log_prob || !entropy || !stats || !dlogits)
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  TokenArgs a = common_args(logits, tokens, wide_tokens, mask, strides, temperature, batch, steps, vocab);
  a.log_prob = const_cast<float*>(log_prob);
  a.entropy = const_cast<float*>(entropy);
  a.stats = const_cast<float*>(stats);
  a.dlog_prob = dlog_prob;
  a.dentropy = dentropy;
  a.dlog_prob_s = RowStride{strides[4], strides[5]};
  a.dentropy_s = RowStride{strides[6], strides[7]};
  a.dlogits = dlogits;
  if (dtype == TOKEN_F32) mask ? launch_bwd<float, true>(as_stream(stream), a) : launch_bwd<float, false>(as_stream(stream), a);
  else mask ? launch_bwd<uint16_t, true>(as_stream(stream), a) : launch_bwd<uint16_t, false>(as_stream(stream), a);
  return check_launch(what);
}
