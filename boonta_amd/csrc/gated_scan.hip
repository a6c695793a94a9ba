// A linear recurrence whose decay and input weight are gated step by step, the
// gates formed in the same pass, and its vector-Jacobian product.
//
// Per feature, with r = sigmoid(decay_gate), i = sigmoid(input_gate):
//   a = exp(-rate r), w = sqrt(1 - a^2), h_t = a_t (done_t ? 0 : h_{t-1}) + w_t i_t x_t
// Backward, from the cotangents g of h and that of the final state:
//   E_t = a'_t (g_t + E_{t+1}) (a' = a, 0 where done; E after the last step: the
//   final state's cotangent; E_0: the carry's), D_t = g_t + E_{t+1},
//   dx = D w i, dinput_gate = D w x i (1 - i), and with
//   dL = D (a h_{t-1} - a^2 i x / w) (h_{t-1} = 0 where done; L = -rate r)
//   ddecay_gate = dL L (1 - r), drate = sum of -dL r.
// 1 - a^2 = -expm1(-2 rate r) is a series where it is small: a^2 rounds away
// there.  A rate of 0 keeps the state: w = 0, and the term through 1 / w is taken as 0.
//
// Sequences of up to SHORT steps are stepped through, a thread for each sequence's
// features.  Else both directions compose affine maps.  A lane holds a chunk of steps of VW
// features in registers, LF lanes stand side by side over the features and the
// rest of the workgroup over the time: a chunk's map, composed with those of the
// chunks before it (lanes by shuffles, waves through LDS), gives the state that
// enters it, and its outputs come from the same registers, so that every operand
// is read once.  Tile follows tile with the state in registers and the next
// tile's operands on their way.  Where sequences and features do not fill the
// chip, the time is cut into segments as well: a launch before forms the map of
// each, and each composes those before it.  The backward forms the states of a
// tile again from the one entering it, which the forward leaves in float32, and
// so needs no output.
//
// A map's decay is -0 where a step of it starts an episode: then nothing of what
// enters, an infinity or NaN neither, passes.
//
// What bounds it: an element takes some 26 vector and 6 transcendental instructions
// forward, about as long as its bytes.  As traced, a launch at a time: 65536 steps of
// 2048 bf16 features, the maps 188 us (4.2 TB/s), the outputs 223 (4.8 TB/s; a copy
// reaches 4.9; untraced both take 388 us together); 256 x 64 steps of 256 float32 features
// 19 us, backward 29 (3.5, 4.0 TB/s); 24 x 4093 of 640 bf16, ragged, 127 and 289 us (3.3, 2.7
// TB/s: the longest sequence's workgroups, one a CU).
#include "row_io.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace ppo;

enum GateDtype { GATE_F32 = 0, GATE_BF16 = 1 };

constexpr int MAX_WAVES = 8;
constexpr int FWD_STEPS = 8, BWD_STEPS = 4, MAP_STEPS = 4;   // of a lane's chunk
constexpr int LANE = 2;                       // features of a lane
constexpr float LOG2E = 1.4426950408889634f;
constexpr int64_t MAX_STRIDE = 1 << 23;       // of a step, in elements: a wave's steps are told apart in 32 bits
constexpr int SHORT = 8;                      // most steps of a short sequence
constexpr int SHORT_THREADS = 256;
constexpr int MAX_SEGMENTS = 256;             // (500000 steps of 64 bf16 features: 64 370 us, 256 114, 512 117)

struct GatedArgs {
  const void *x, *input_gate, *decay_gate;
  const float* rate;
  const float* carry;       // [batch, F], or null (zeros)
  const uint8_t* done;      // [batch, steps], or null
  const int32_t* lengths;   // [batch], or null (steps)
  void* out;                // forward
  float* final;
  float* states;            // [batch, saved, F], entering every `save`-th step
  float* maps;              // [batch, segments, 2, F]: decay, sum
  const void* dout;         // backward
  const float* dfinal;      // or null (zeros)
  void *dx, *dinput_gate, *ddecay_gate;
  float* dcarry;            // or null
  float* partials;          // [batch, segments, F]: drate, or null
  RowStride x_s, input_s, decay_s, dout_s;
  int steps, F, blocks;     // blocks: workgroups over the features
  int segment, segments;    // steps of one; how many
  int save_log2, saved;
};

__device__ __forceinline__ bool is_reset(float a) { return __float_as_uint(a) == 0x80000000u; }
// The map (a, b) of h; b alone past a reset.
__device__ __forceinline__ float apply(float a, float b, float h) { return is_reset(a) ? b : __fmaf_rn(a, h, b); }
// The decay of two maps one after the other.
__device__ __forceinline__ float decay_of(float later, float earlier) { return is_reset(later) ? later : later * earlier; }

struct Gates {
  float a, wi;                // decay; w i
  float i, r, not_i, not_r;   // not_: 1 - it
  float over_w;               // 1 / w; 0 where w is (the hardware's root of a subnormal number is 0)
};
// 1 - a^2 of a = 2^-q.  Below 2 ln(2) q = 1/8 the Chebyshev interpolation of degree 3 of
// (1 - 2^-2q) / q, within 2^-25 of it; above, what the difference loses is at most 8 times a^2's rounding.
__device__ __forceinline__ float one_minus_square(float a, float q) {
  float s = __fmaf_rn(q, -0.1464114f, 0.44361513f);
  s = __fmaf_rn(q, s, -0.96089852f);
  s = __fmaf_rn(q, s, 1.38629434f);
  return q < 0.0901684f ? q * s : __fmaf_rn(-a, a, 1.f);
}
// rl = rate log2(e).  BWD: what the gradients need too.
template <bool BWD> __device__ __forceinline__ Gates gates_of(float input, float decay, float rl) {
  Gates g;
  g.i = sigmoid(input, g.not_i);
  g.r = sigmoid(decay, g.not_r);
  const float q = rl * g.r;
  g.a = __builtin_amdgcn_exp2f(-q);
  const float w2 = one_minus_square(g.a, q);
  if constexpr (BWD) {
    g.over_w = w2 >= 1.17549435e-38f ? __builtin_amdgcn_rsqf(w2) : 0.f;   // (of a subnormal number it is infinite)
    g.wi = w2 * g.over_w * g.i;
  } else {
    g.wi = __builtin_amdgcn_sqrtf(w2) * g.i;
  }
  return g;
}

// VW values as stored.
template <typename S, int VW> struct Raw {
  S v[VW];
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
template <typename S, int VW> __device__ __forceinline__ Raw<S, VW> load_raw(const char* base, int64_t offset) {
  Raw<S, VW> r;
  __builtin_memcpy(r.v, base + offset, sizeof(r.v));
  return r;
}
// (a base of the whole wave and a lane's 32-bit offset)
template <typename S, int VW> __device__ __forceinline__ Raw<S, VW> load_near(const char* base, uint32_t offset) {
  Raw<S, VW> r;
  __builtin_memcpy(r.v, base + offset, sizeof(r.v));
  return r;
}
template <int VW> __device__ __forceinline__ void store_near(float* base, uint32_t offset, const float (&v)[VW]) {
  __builtin_memcpy(reinterpret_cast<char*>(base) + offset, v, 4 * VW);
}
template <int VW> __device__ __forceinline__ void store_near(uint16_t* base, uint32_t offset, const float (&v)[VW]) {
  char* p = reinterpret_cast<char*>(base) + offset;
  if constexpr (VW == 1) {
    const uint16_t u = (uint16_t)pack_bf16(v[0], v[0]);
    __builtin_memcpy(p, &u, 2);
  } else {
    uint32_t u[VW / 2];
#pragma unroll
    for (int k = 0; k < VW / 2; ++k) u[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
    __builtin_memcpy(p, u, 2 * VW);
  }
}

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Flags of up to 8 steps from t on (those below `steps`), a byte each.
template <int N> __device__ __forceinline__ uint64_t load_flags(const uint8_t* done, int t, int steps) {
  uint64_t f = 0;
  if (t + N <= steps) {
    __builtin_memcpy(&f, done + t, N);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (t + i < steps) f |= (uint64_t)done[t + i] << (8 * i);
  }
  return f;
}
__device__ __forceinline__ bool flag(uint64_t f, int i) { return (f >> (8 * i)) & 0xff; }

// Where a lane stands: LF lanes over the features, SLOTS of a wave over the
// time, each with a chunk of N steps.
template <int VW, int LF, int N> struct Lane {
  static constexpr int SLOTS = 64 / LF;
  int lane, wave, waves, slot, b, f0, tile;
  __device__ __forceinline__ explicit Lane(const GatedArgs& p) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    waves = blockDim.x >> 6;
    slot = lane / LF;
    b = blockIdx.x / p.blocks;
    const int fb = blockIdx.x - b * p.blocks;
    // lanes past the row's end repeat its last features: they read and write the same values
    f0 = min((fb * LF + lane % LF) * VW, p.F - VW);
    tile = waves * SLOTS * N;
  }
  // first step of the wave's, and the lane's, chunks in the tile from t0 on
  __device__ __forceinline__ int wave_step(int t0) const { return t0 + wave * SLOTS * N; }
  __device__ __forceinline__ int chunk_step(int t0) const { return wave_step(t0) + slot * N; }
};

// In a branch that is seldom taken: at its head, its instructions are not formed
// beside the other's and selected from (which took a fifth of the loop's); at
// its end, its loads stay its own (joined with the other's they take 64-bit addresses).
__device__ __forceinline__ void apart() { asm volatile(""); }

// A tensor's N steps of a lane's chunk: row offsets within 32 bits of the
// wave's first where the tile is whole, clamped rows of it otherwise.
template <typename S, int VW, int N, typename L>
__device__ __forceinline__ void fetch_steps(const void* x, const RowStride& s, const L& at, int t0, int end, bool whole,
                                            Raw<S, VW> (&v)[N]) {
  const char* base = static_cast<const char*>(x) + (int64_t)at.b * s.batch * (int64_t)sizeof(S);
  if (whole) {
    const uint32_t near = (uint32_t)(at.slot * N * (int)s.step + at.f0) * (uint32_t)sizeof(S);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = load_near<S, VW>(base + (at.wave_step(t0) + i) * s.step * (int64_t)sizeof(S), near);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = load_raw<S, VW>(base, (min(at.chunk_step(t0) + i, end - 1) * s.step + at.f0) * (int64_t)sizeof(S));
    apart();
  }
}
// and of an output [batch, steps, F]: steps below `end`.
template <typename S, int VW, int N, typename L>
__device__ __forceinline__ void store_step(void* out, const GatedArgs& p, const L& at, int t0, int i, int end, bool whole,
                                           const float (&v)[VW]) {
  if (!whole && at.chunk_step(t0) + i >= end) return;
  S* base = static_cast<S*>(out) + ((int64_t)at.b * p.steps + at.wave_step(t0) + i) * p.F;
  store_near<VW>(base, (uint32_t)(at.slot * N * p.F + at.f0) * (uint32_t)sizeof(S), v);
}
template <typename S, int VW, int LF, int N>
__device__ __forceinline__ void clear_steps(void* out, const GatedArgs& p, const Lane<VW, LF, N>& at, int from, int end) {
  float zero[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) zero[k] = 0.f;
  for (int t = from + at.wave * at.SLOTS + at.slot; t < end; t += at.waves * at.SLOTS)
    store_near<VW>(static_cast<S*>(out) + ((int64_t)at.b * p.steps + t) * p.F, (uint32_t)at.f0 * (uint32_t)sizeof(S), zero);
}

// The state of VW features at b's row of a [batch, F] array, or zeros.
template <int VW> __device__ __forceinline__ void load_state(const float* p, int64_t at, float (&h)[VW]) {
#pragma unroll
  for (int k = 0; k < VW; ++k) h[k] = p ? p[at + k] : 0.f;
}

// The maps (A, B) of a wave's slots composed: on return those of the slots
// before (REVERSE: after) the lane's, and in LDS the wave's own.
template <int VW, int LF, bool REVERSE>
__device__ __forceinline__ void compose_slots(float (&A)[VW], float (&B)[VW], int lane, float* wave_a, float* wave_b) {
  constexpr int SLOTS = 64 / LF;
  const int slot = REVERSE ? SLOTS - 1 - lane / LF : lane / LF;   // (in the order of the maps)
#pragma unroll
  for (int d = 1; d < SLOTS; d <<= 1) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      const int from = REVERSE ? lane + d * LF : lane - d * LF;
      const float a = __shfl(A[k], from), b = __shfl(B[k], from);
      if (slot >= d) {
        B[k] = apply(A[k], B[k], b);
        A[k] = decay_of(A[k], a);
      }
    }
  }
  if (slot == SLOTS - 1) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      wave_a[(lane % LF) * VW + k] = A[k];
      wave_b[(lane % LF) * VW + k] = B[k];
    }
  }
  if constexpr (SLOTS > 1) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      const int from = REVERSE ? lane + LF : lane - LF;
      const float a = __shfl(A[k], from), b = __shfl(B[k], from);
      A[k] = slot > 0 ? a : 1.f;
      B[k] = slot > 0 ? b : 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      A[k] = 1.f;
      B[k] = 0.f;
    }
  }
}
// The state h entering the tile carried through the waves' maps: on return h
// leaves the tile, and `mine` enters the lane's chunk, whose slots' map before it is (A, B).
template <int VW, int LF, bool REVERSE>
__device__ __forceinline__ void through_waves(float (&h)[VW], float (&mine)[VW], const float (&A)[VW],
                                              const float (&B)[VW], const float* wave_a, const float* wave_b, int lane,
                                              int wave, int waves) {
  const auto step = [&](int w, const float (&a)[VW], const float (&b)[VW]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      mine[k] = w == wave ? h[k] : mine[k];
      h[k] = apply(a[k], b[k], h[k]);
    }
  };
  const auto read = [&](int w, float (&a)[VW], float (&b)[VW]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      a[k] = wave_a[(w * LF + lane % LF) * VW + k];
      b[k] = wave_b[(w * LF + lane % LF) * VW + k];
    }
  };
#pragma unroll
  for (int k = 0; k < VW; ++k) mine[k] = h[k];
  if (waves == MAX_WAVES) {   // (half of the reads on their way at once)
    constexpr int H = MAX_WAVES / 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float a[H][VW], b[H][VW];
#pragma unroll
      for (int i = 0; i < H; ++i) read(REVERSE ? MAX_WAVES - 1 - half * H - i : half * H + i, a[i], b[i]);
#pragma unroll
      for (int i = 0; i < H; ++i) step(REVERSE ? MAX_WAVES - 1 - half * H - i : half * H + i, a[i], b[i]);
    }
  } else {
    for (int i = 0; i < waves; ++i) {
      const int w = REVERSE ? waves - 1 - i : i;
      float a[VW], b[VW];
      read(w, a, b);
      step(w, a, b);
    }
  }
#pragma unroll
  for (int k = 0; k < VW; ++k) mine[k] = apply(A[k], B[k], mine[k]);
}

// The state h carried through the segments before (REVERSE: after) this one: a run of
// their maps for each slot, composed as the chunks of a tile are (65536 steps of 64
// bf16 features in 64 segments 54 us, every lane reading them all 60).  Rooms of LDS
// that the first tile does not use.
template <int VW, int LF, bool REVERSE, typename L>
__device__ __forceinline__ void through_segments(const GatedArgs& p, const L& at, int segment, float (&h)[VW],
                                                 float* wave_a, float* wave_b) {
  if (p.segments == 1) return;
  const int n = REVERSE ? p.segments - 1 - segment : segment, slots = at.waves * at.SLOTS;
  const int slot = at.wave * at.SLOTS + at.slot, each = (n + slots - 1) / slots;
  const int first = (REVERSE ? slots - 1 - slot : slot) * each;
  float A[VW], B[VW], mine[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    A[k] = 1.f;
    B[k] = 0.f;
  }
  constexpr int U = 4;   // maps on their way at once
  for (int i0 = 0; i0 < each; i0 += U) {
    float a[U][VW], s[U][VW];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(first + i0 + u, n - 1);
      const float* m = p.maps + (((int64_t)at.b * p.segments + (REVERSE ? p.segments - 1 - i : i)) * 2) * p.F + at.f0;
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        a[u][k] = m[k];
        s[u][k] = m[p.F + k];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = i0 + u < each && first + i0 + u < n;
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        B[k] = there ? apply(a[u][k], s[u][k], B[k]) : B[k];
        A[k] = there ? decay_of(a[u][k], A[k]) : A[k];
      }
    }
  }
  compose_slots<VW, LF, REVERSE>(A, B, at.lane, wave_a + at.wave * LF * VW, wave_b + at.wave * LF * VW);
  lds_barrier();
  through_waves<VW, LF, REVERSE>(h, mine, A, B, wave_a, wave_b, at.lane, at.wave, at.waves);
}

// The map of a segment: of the state h (REVERSE: of the cotangent E).  Every
// slot takes a part of the segment's steps from one end to the other, and the
// parts are composed at the end.
template <typename S, int VW, int LF, bool REVERSE>
__global__ void __launch_bounds__(64 * MAX_WAVES) gated_maps_kernel(GatedArgs p) {
  constexpr int N = MAP_STEPS;
  __shared__ float wave_a[MAX_WAVES * LF * VW], wave_b[MAX_WAVES * LF * VW];
  const Lane<VW, LF, N> at(p);
  const int segment = blockIdx.y + (REVERSE ? 1 : 0), begin = segment * p.segment;   // (the first, or last, needs none)
  const int end = min(p.steps, begin + p.segment);
  const int live_end = min(end, p.lengths ? max(0, min(p.lengths[at.b], p.steps)) : p.steps);
  const uint8_t* done = p.done ? p.done + (int64_t)at.b * p.steps : nullptr;
  const int part = p.segment / (at.waves * at.SLOTS);   // steps of a slot, a multiple of N
  const int wave_first = begin + at.wave * at.SLOTS * part, first = wave_first + at.slot * part;
  const int wave_last = wave_first + (at.SLOTS - 1) * part;
  float A[VW], B[VW], rl[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    rl[k] = p.rate[at.f0 + k] * LOG2E;
    A[k] = 1.f;
    B[k] = 0.f;
  }
  Raw<S, VW> x[N], ig[N], dg[N];   // of the next chunk (REVERSE: x the cotangent, no ig)
  uint64_t flags = 0;
  auto load = [&](const void* from, const RowStride& s, int c, Raw<S, VW>(&v)[N]) __attribute__((always_inline)) {
    const char* base = static_cast<const char*>(from) + (int64_t)at.b * s.batch * (int64_t)sizeof(S);
    const int t = first + c;
    if (wave_last + c + N <= live_end) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (at.SLOTS == 1)
          v[i] = load_near<S, VW>(base + (wave_first + c + i) * s.step * (int64_t)sizeof(S), (uint32_t)at.f0 * (uint32_t)sizeof(S));
        else
          v[i] = load_raw<S, VW>(base, ((t + i) * s.step + at.f0) * (int64_t)sizeof(S));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = load_raw<S, VW>(base, (min(t + i, live_end - 1) * s.step + at.f0) * (int64_t)sizeof(S));
      apart();
    }
  };
  auto fetch = [&](int c) __attribute__((always_inline)) {
    load(p.decay_gate, p.decay_s, c, dg);
    load(REVERSE ? p.dout : p.x, REVERSE ? p.dout_s : p.x_s, c, x);
    if constexpr (!REVERSE) load(p.input_gate, p.input_s, c, ig);
    if (done) flags = load_flags<N>(done, first + c, p.steps);
  };
  // chunks of the wave's first slot that has the most live steps
  const int chunks = (max(0, min(part, live_end - wave_first)) + N - 1) / N;
  if (chunks > 0) fetch(REVERSE ? (chunks - 1) * N : 0);
  for (int j = 0; j < chunks; ++j) {
    const int c = (REVERSE ? chunks - 1 - j : j) * N;
    float a[N][VW], b[N][VW];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Gates g = gates_of<false>(REVERSE ? 0.f : widen(ig[i].v[k]), widen(dg[i].v[k]), rl[k]);
        a[i][k] = g.a;
        b[i][k] = REVERSE ? widen(x[i].v[k]) : g.wi * widen(x[i].v[k]);
      }
    const uint64_t cuts = flags;
    if (j + 1 < chunks) fetch(REVERSE ? c - N : c + N);
    if (__any(cuts != 0) || wave_last + c + N > live_end) {
      apart();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = REVERSE ? N - 1 - i : i;
        const bool live = first + c + e < live_end, cut = flag(cuts, e);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const float ae = live ? (cut ? -0.f : a[e][k]) : 1.f, be = live ? b[e][k] : 0.f;
          B[k] = REVERSE ? (is_reset(ae) ? 0.f : ae * (be + B[k])) : apply(ae, be, B[k]);
          A[k] = decay_of(ae, A[k]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = REVERSE ? N - 1 - i : i;
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          B[k] = REVERSE ? a[e][k] * (b[e][k] + B[k]) : __fmaf_rn(a[e][k], B[k], b[e][k]);
          A[k] *= a[e][k];
        }
      }
    }
  }
  compose_slots<VW, LF, REVERSE>(A, B, at.lane, wave_a + at.wave * LF * VW, wave_b + at.wave * LF * VW);
  __syncthreads();
  if (at.wave > 0 || at.slot > 0) return;
  float decay[VW], sum[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    decay[k] = 1.f;
    sum[k] = 0.f;
  }
  for (int i = 0; i < at.waves; ++i) {
    const int w = REVERSE ? at.waves - 1 - i : i;
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      const int j = (w * LF + at.lane) * VW + k;
      sum[k] = apply(wave_a[j], wave_b[j], sum[k]);
      decay[k] = decay_of(wave_a[j], decay[k]);
    }
  }
  float* m = p.maps + (((int64_t)at.b * p.segments + segment) * 2) * p.F + at.f0;
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    m[k] = decay[k];
    m[p.F + k] = sum[k];
  }
}

template <typename S, int VW, int LF>
__global__ void __launch_bounds__(64 * MAX_WAVES) gated_fwd_kernel(GatedArgs p) {
  constexpr int N = FWD_STEPS;
  __shared__ float wave_a[2][MAX_WAVES * LF * VW], wave_b[2][MAX_WAVES * LF * VW];
  const Lane<VW, LF, N> at(p);
  const int segment = blockIdx.y, begin = segment * p.segment, end = min(p.steps, begin + p.segment);
  const int live_end = min(end, p.lengths ? max(0, min(p.lengths[at.b], p.steps)) : p.steps);
  const uint8_t* done = p.done ? p.done + (int64_t)at.b * p.steps : nullptr;
  float h[VW], rl[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) rl[k] = p.rate[at.f0 + k] * LOG2E;
  Raw<S, VW> x[N], ig[N], dg[N];   // of the next tile
  uint64_t flags = 0;
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    const bool whole = t0 + at.tile <= live_end;
    fetch_steps<S, VW, N>(p.x, p.x_s, at, t0, live_end, whole, x);
    fetch_steps<S, VW, N>(p.input_gate, p.input_s, at, t0, live_end, whole, ig);
    fetch_steps<S, VW, N>(p.decay_gate, p.decay_s, at, t0, live_end, whole, dg);
    if (done) flags = load_flags<N>(done, at.chunk_step(t0), p.steps);
  };
  if (begin < live_end) fetch(begin);
  load_state<VW>(p.carry, (int64_t)at.b * p.F + at.f0, h);
  through_segments<VW, LF, false>(p, at, segment, h, wave_a[1], wave_b[1]);
  int set = 0, t0 = begin;
  for (; t0 < live_end; t0 += at.tile, set ^= 1) {
    const bool whole = t0 + at.tile <= live_end;
    const int t = at.chunk_step(t0);
    const bool resets = __any(flags != 0);
    float a[N][VW], b[N][VW], A[VW], B[VW], mine[VW];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Gates g = gates_of<false>(widen(ig[i].v[k]), widen(dg[i].v[k]), rl[k]);
        a[i][k] = g.a;
        b[i][k] = g.wi * widen(x[i].v[k]);
      }
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      A[k] = 1.f;
      B[k] = 0.f;
    }
    if (resets || !whole) {
      apart();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool live = t + i < live_end, cut = flag(flags, i);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          a[i][k] = live ? (cut ? -0.f : a[i][k]) : 1.f;
          b[i][k] = live ? b[i][k] : 0.f;
          B[k] = apply(a[i][k], b[i][k], B[k]);
          A[k] = decay_of(a[i][k], A[k]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          B[k] = __fmaf_rn(a[i][k], B[k], b[i][k]);
          A[k] *= a[i][k];
        }
    }
    if (t0 + at.tile < live_end) fetch(t0 + at.tile);
    float *pa = wave_a[set], *pb = wave_b[set];
    compose_slots<VW, LF, false>(A, B, at.lane, pa + at.wave * LF * VW, pb + at.wave * LF * VW);
    lds_barrier();
    through_waves<VW, LF, false>(h, mine, A, B, pa, pb, at.lane, at.wave, at.waves);
    if (p.states && t < live_end && (t & ((1 << p.save_log2) - 1)) == 0) {
      float* s = p.states + ((int64_t)at.b * p.saved + (t >> p.save_log2)) * p.F + at.f0;
#pragma unroll
      for (int k = 0; k < VW; ++k) s[k] = mine[k];
    }
    if (resets || !whole) {
    apart();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float o[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          mine[k] = apply(a[i][k], b[i][k], mine[k]);
          o[k] = t + i < live_end ? mine[k] : 0.f;
        }
        store_step<S, VW, N>(p.out, p, at, t0, i, end, whole, o);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int k = 0; k < VW; ++k) mine[k] = __fmaf_rn(a[i][k], mine[k], b[i][k]);
        store_step<S, VW, N>(p.out, p, at, t0, i, end, true, mine);
      }
    }
  }
  clear_steps<S>(p.out, p, at, t0, end);
  if (segment == p.segments - 1 && at.wave == 0 && at.slot == 0) {
    float* f = p.final + (int64_t)at.b * p.F + at.f0;
#pragma unroll
    for (int k = 0; k < VW; ++k) f[k] = h[k];
  }
}

// What the backward keeps of an element while the maps are composed.
struct Kept {
  float a, b, g;        // decay (-0 at a reset, 1 past the end), input, cotangent
  float wi, not_i, c;   // w i; 1 - i; a^2 i x / w
  float r, not_r;       // and 1 - r
};
__device__ __forceinline__ Kept kept_of(const Gates& g, float x, float cotangent) {
  return Kept{g.a, g.wi * x, cotangent, g.wi, g.not_i, g.a * g.over_w * g.a * (g.i * x), g.r, g.not_r};
}

template <typename S, int VW, int LF>
__global__ void __launch_bounds__(64 * MAX_WAVES) gated_bwd_kernel(GatedArgs p) {
  constexpr int N = BWD_STEPS;
  __shared__ float fwd_a[2][MAX_WAVES * LF * VW], fwd_b[2][MAX_WAVES * LF * VW];
  __shared__ float rev_a[2][MAX_WAVES * LF * VW], rev_b[2][MAX_WAVES * LF * VW];
  const Lane<VW, LF, N> at(p);
  const int segment = blockIdx.y, begin = segment * p.segment, end = min(p.steps, begin + p.segment);
  const int live_end = min(end, p.lengths ? max(0, min(p.lengths[at.b], p.steps)) : p.steps);
  const uint8_t* done = p.done ? p.done + (int64_t)at.b * p.steps : nullptr;
  const int64_t state = (int64_t)at.b * p.F + at.f0;
  float E[VW], rate[VW], rl[VW], drate[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    rate[k] = p.rate[at.f0 + k];
    rl[k] = rate[k] * LOG2E;
    drate[k] = 0.f;
  }
  Raw<S, VW> x[N], ig[N], dg[N], go[N];   // of the tile before
  float entering[VW];
  uint64_t flags = 0;
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    const bool whole = t0 + at.tile <= live_end;
    fetch_steps<S, VW, N>(p.decay_gate, p.decay_s, at, t0, live_end, whole, dg);
    fetch_steps<S, VW, N>(p.dout, p.dout_s, at, t0, live_end, whole, go);
    fetch_steps<S, VW, N>(p.x, p.x_s, at, t0, live_end, whole, x);
    fetch_steps<S, VW, N>(p.input_gate, p.input_s, at, t0, live_end, whole, ig);
    load_state<VW>(p.states, ((int64_t)at.b * p.saved + (t0 >> p.save_log2)) * p.F + at.f0, entering);
    if (done) flags = load_flags<N>(done, at.chunk_step(t0), p.steps);
  };
  const int tiles = live_end > begin ? (live_end - begin + at.tile - 1) / at.tile : 0;
  int set = 0, t0 = begin + (tiles - 1) * at.tile;
  if (tiles > 0) fetch(t0);
  load_state<VW>(p.dfinal, state, E);
  through_segments<VW, LF, true>(p, at, segment, E, rev_a[1], rev_b[1]);
  for (; t0 >= begin; t0 -= at.tile, set ^= 1) {
    const bool whole = t0 + at.tile <= live_end;
    const int t = at.chunk_step(t0);
    const bool resets = __any(flags != 0);
    Kept q[N][VW];
    float h[VW], A[VW], B[VW], RA[VW], RB[VW];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Gates g = gates_of<true>(widen(ig[i].v[k]), widen(dg[i].v[k]), rl[k]);
        q[i][k] = kept_of(g, widen(x[i].v[k]), widen(go[i].v[k]));
      }
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      A[k] = RA[k] = 1.f;
      B[k] = RB[k] = 0.f;
      h[k] = entering[k];
    }
    if (resets || !whole) {
      apart();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool live = t + i < live_end, cut = flag(flags, i);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          Kept& e = q[i][k];
          e.a = live ? (cut ? -0.f : e.a) : 1.f;
          e.b = live ? e.b : 0.f;
          e.g = live ? e.g : 0.f;
          B[k] = apply(e.a, e.b, B[k]);
          A[k] = decay_of(e.a, A[k]);
        }
      }
      // (the cotangents' map in its own order: a NaN decay behind a reset, multiplied to it, is no reset)
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          RB[k] = is_reset(q[i][k].a) ? 0.f : q[i][k].a * (q[i][k].g + RB[k]);
          RA[k] = decay_of(q[i][k].a, RA[k]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          B[k] = __fmaf_rn(q[i][k].a, B[k], q[i][k].b);
          A[k] *= q[i][k].a;
          RB[k] = q[N - 1 - i][k].a * (q[N - 1 - i][k].g + RB[k]);
        }
#pragma unroll
      for (int k = 0; k < VW; ++k) RA[k] = A[k];
    }
    if (t0 > begin) fetch(t0 - at.tile);
    const int mine_at = at.wave * LF * VW;
    compose_slots<VW, LF, false>(A, B, at.lane, fwd_a[set] + mine_at, fwd_b[set] + mine_at);
    compose_slots<VW, LF, true>(RA, RB, at.lane, rev_a[set] + mine_at, rev_b[set] + mine_at);
    lds_barrier();
    float mine[VW], after[VW], before[N][VW];
    through_waves<VW, LF, false>(h, mine, A, B, fwd_a[set], fwd_b[set], at.lane, at.wave, at.waves);
    through_waves<VW, LF, true>(E, after, RA, RB, rev_a[set], rev_b[set], at.lane, at.wave, at.waves);
    if (resets) {
      apart();
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          before[i][k] = is_reset(q[i][k].a) ? 0.f : mine[k];
          mine[k] = apply(q[i][k].a, q[i][k].b, mine[k]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          before[i][k] = mine[k];
          mine[k] = __fmaf_rn(q[i][k].a, mine[k], q[i][k].b);
        }
    }
    auto gradients = [&](auto plain) __attribute__((always_inline)) {   // no resets, a whole tile
      constexpr bool PLAIN = decltype(plain)::value;
      if constexpr (!PLAIN) apart();
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        const bool live = PLAIN || t + i < live_end;
        float ox[VW], oi[VW], od[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const Kept& e = q[i][k];
          const float D = e.g + after[k];
          after[k] = !PLAIN && is_reset(e.a) ? 0.f : e.a * D;
          const float dr = D * __fmaf_rn(e.a, before[i][k], -e.c) * e.r;   // dL r
          ox[k] = live ? D * e.wi : 0.f;
          oi[k] = live ? D * e.b * e.not_i : 0.f;
          od[k] = live ? -dr * rate[k] * e.not_r : 0.f;
          drate[k] -= live ? dr : 0.f;
        }
        store_step<S, VW, N>(p.dx, p, at, t0, i, end, whole, ox);
        store_step<S, VW, N>(p.dinput_gate, p, at, t0, i, end, whole, oi);
        store_step<S, VW, N>(p.ddecay_gate, p, at, t0, i, end, whole, od);
      }
    };
    if (resets || !whole) gradients(std::false_type{});
    else gradients(std::true_type{});
  }
  const int cleared = begin + tiles * at.tile;
  clear_steps<S>(p.dx, p, at, cleared, end);
  clear_steps<S>(p.dinput_gate, p, at, cleared, end);
  clear_steps<S>(p.ddecay_gate, p, at, cleared, end);
  if (p.dcarry && segment == 0 && at.wave == 0 && at.slot == 0) {
#pragma unroll
    for (int k = 0; k < VW; ++k) p.dcarry[state + k] = E[k];
  }
  if (p.partials) {
    // the slots' sums, the lanes' by butterflies, the waves' in their order
    float* sums = &fwd_a[0][0];
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      for (int o = LF; o < 64; o <<= 1) drate[k] += __shfl_xor(drate[k], o);
    }
    __syncthreads();
    if (at.slot == 0) {
#pragma unroll
      for (int k = 0; k < VW; ++k) sums[(at.wave * LF + at.lane) * VW + k] = drate[k];
    }
    __syncthreads();
    if (at.wave == 0 && at.slot == 0) {
      float* out = p.partials + ((int64_t)at.b * p.segments + segment) * p.F + at.f0;
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        float s = 0.f;
        for (int w = 0; w < at.waves; ++w) s += sums[(w * LF + at.lane) * VW + k];
        out[k] = s;
      }
    }
  }
}

// ---- short sequences: a thread takes VW features through all steps of a sequence and
// goes on to the next, with no exchange, and is bound by HBM: 33M bf16 elements in
// sequences of one step take 106 us (5.0 TB/s), in chunks 484; of four 66 for 133, of
// eight 57 for 65; both passes 312, 197, 195 us (4.5 to 4.2 TB/s) for 1583, 410, 228.
// Its lanes stand side by side over the features, the rest of the workgroup over
// the sequences.
template <int VW> struct ShortLane {
  int lane, row, rows, f0;
  __device__ __forceinline__ ShortLane(const GatedArgs& p, int lanes_log2) {
    lane = threadIdx.x & ((1 << lanes_log2) - 1);
    row = threadIdx.x >> lanes_log2;
    rows = SHORT_THREADS >> lanes_log2;
    // (lanes past the row's end repeat its last features: they read and write the same values)
    f0 = min((int)((blockIdx.x << lanes_log2) + lane) * VW, p.F - VW);
  }
};
// A sequence's steps of an operand, the last again where there are fewer than N.
template <typename S, int VW, int N>
__device__ __forceinline__ void fetch_short(const void* x, const RowStride& s, const GatedArgs& p, int64_t b, int f0,
                                            Raw<S, VW> (&v)[N]) {
  const char* base = static_cast<const char*>(x);
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = load_raw<S, VW>(base, (b * s.batch + min(i, p.steps - 1) * s.step + f0) * (int64_t)sizeof(S));
}
template <int N> __device__ __forceinline__ uint32_t short_flags(const GatedArgs& p, int64_t b) {
  uint32_t cuts = 0;
  if (p.done) {
#pragma unroll
    for (int i = 0; i < N; ++i) cuts |= (p.done[b * p.steps + min(i, p.steps - 1)] ? 1u : 0u) << i;
  }
  return cuts;
}
template <typename S, int VW> __device__ __forceinline__ void store_short(void* out, int64_t at, const float (&v)[VW]) {
  store_near<VW>(static_cast<S*>(out) + at, 0, v);
}

template <typename S, int VW, int N>
__global__ void __launch_bounds__(SHORT_THREADS) gated_short_fwd_kernel(GatedArgs p, int batch, int lanes_log2) {
  const ShortLane<VW> at(p, lanes_log2);
  float rl[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) rl[k] = p.rate[at.f0 + k] * LOG2E;
  for (int64_t b = (int64_t)blockIdx.y * at.rows + at.row; b < batch; b += (int64_t)gridDim.y * at.rows) {
    Raw<S, VW> x[N], ig[N], dg[N];
    fetch_short<S, VW, N>(p.x, p.x_s, p, b, at.f0, x);
    fetch_short<S, VW, N>(p.input_gate, p.input_s, p, b, at.f0, ig);
    fetch_short<S, VW, N>(p.decay_gate, p.decay_s, p, b, at.f0, dg);
    const uint32_t cuts = short_flags<N>(p, b);
    const int live_end = p.lengths ? max(0, min(p.lengths[b], p.steps)) : p.steps;
    float h[VW];
    load_state<VW>(p.carry, b * p.F + at.f0, h);
    if (p.states) store_near<VW>(p.states + b * p.F + at.f0, 0, h);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= p.steps) break;
      const bool live = i < live_end, cut = cuts >> i & 1;
      float o[VW];
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Gates g = gates_of<false>(widen(ig[i].v[k]), widen(dg[i].v[k]), rl[k]);
        const float next = apply(cut ? -0.f : g.a, g.wi * widen(x[i].v[k]), h[k]);
        h[k] = live ? next : h[k];
        o[k] = live ? next : 0.f;
      }
      store_short<S, VW>(p.out, (b * p.steps + i) * p.F + at.f0, o);
    }
    store_near<VW>(p.final + b * p.F + at.f0, 0, h);
  }
}

template <typename S, int VW, int N>
__global__ void __launch_bounds__(SHORT_THREADS) gated_short_bwd_kernel(GatedArgs p, int batch, int lanes_log2) {
  __shared__ float sums[SHORT_THREADS * VW];
  const ShortLane<VW> at(p, lanes_log2);
  float rate[VW], rl[VW], drate[VW];
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    rate[k] = p.rate[at.f0 + k];
    rl[k] = rate[k] * LOG2E;
    drate[k] = 0.f;
  }
  for (int64_t b = (int64_t)blockIdx.y * at.rows + at.row; b < batch; b += (int64_t)gridDim.y * at.rows) {
    Raw<S, VW> x[N], ig[N], dg[N], go[N];
    fetch_short<S, VW, N>(p.x, p.x_s, p, b, at.f0, x);
    fetch_short<S, VW, N>(p.input_gate, p.input_s, p, b, at.f0, ig);
    fetch_short<S, VW, N>(p.decay_gate, p.decay_s, p, b, at.f0, dg);
    fetch_short<S, VW, N>(p.dout, p.dout_s, p, b, at.f0, go);
    const uint32_t cuts = short_flags<N>(p, b);
    const int live_end = p.lengths ? max(0, min(p.lengths[b], p.steps)) : p.steps;
    float h[VW], E[VW], before[N][VW];
    load_state<VW>(p.states, b * p.F + at.f0, h);
    load_state<VW>(p.dfinal, b * p.F + at.f0, E);
    Kept q[N][VW];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Gates g = gates_of<true>(widen(ig[i].v[k]), widen(dg[i].v[k]), rl[k]);
        const float xv = widen(x[i].v[k]);
        const bool cut = cuts >> i & 1;
        q[i][k] = kept_of(g, xv, widen(go[i].v[k]));
        if (cut) q[i][k].a = -0.f;
        before[i][k] = cut ? 0.f : h[k];
        h[k] = i < live_end ? apply(q[i][k].a, q[i][k].b, h[k]) : h[k];
      }
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
      if (i >= p.steps) continue;
      const bool live = i < live_end;
      float ox[VW], oi[VW], od[VW];
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const Kept& e = q[i][k];
        const float D = e.g + E[k];
        const float dr = D * __fmaf_rn(e.a, before[i][k], -e.c) * e.r;   // dL r
        E[k] = live ? (is_reset(e.a) ? 0.f : e.a * D) : E[k];
        ox[k] = live ? D * e.wi : 0.f;
        oi[k] = live ? D * e.b * e.not_i : 0.f;
        od[k] = live ? -dr * rate[k] * e.not_r : 0.f;
        drate[k] -= live ? dr : 0.f;
      }
      const int64_t to = (b * p.steps + i) * p.F + at.f0;
      store_short<S, VW>(p.dx, to, ox);
      store_short<S, VW>(p.dinput_gate, to, oi);
      store_short<S, VW>(p.ddecay_gate, to, od);
    }
    if (p.dcarry) store_near<VW>(p.dcarry + b * p.F + at.f0, 0, E);
  }
  if (!p.partials) return;
#pragma unroll
  for (int k = 0; k < VW; ++k) sums[k * SHORT_THREADS + threadIdx.x] = drate[k];
  __syncthreads();
  if (at.row > 0) return;
#pragma unroll
  for (int k = 0; k < VW; ++k) {
    float s = 0.f;
    for (int r = 0; r < at.rows; ++r) s += sums[k * SHORT_THREADS + (r << lanes_log2) + at.lane];
    p.partials[(int64_t)blockIdx.y * p.F + at.f0 + k] = s;
  }
}

// Sums over rows [from, from + each) of parts [rows, F]: 64 columns a workgroup,
// each wave its share of the rows in their order, then the waves'.
__global__ void __launch_bounds__(1024) gated_rate_kernel(const float* parts, int64_t rows, int each, int F, float* out) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, f = blockIdx.x * 64 + lane;
  const int64_t from = (int64_t)blockIdx.y * each, to = min(rows, from + each);
  const int share = (each + 15) / 16;
  const int64_t b1 = min(to, from + (int64_t)(wave + 1) * share);
  float s = 0.f;
  if (f < F) {
    for (int64_t b0 = from + (int64_t)wave * share; b0 < b1; b0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = parts[min(b0 + k, b1 - 1) * F + f];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += b0 + k < b1 ? v[k] : 0.f;
    }
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || f >= F) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += sums[w][lane];
  out[(int64_t)blockIdx.y * F + f] = s;
}

// One step (64 x 1000 bf16 features 3.2 us, a launch and its loads' latency): a thread
// for VW features of a sequence, fewer at the row's end (the
// new state may be the old one's memory, so that each is read by its writer alone).
template <typename S, int VW>
__global__ void __launch_bounds__(256) gated_step_kernel(GatedArgs p, int64_t threads, int per_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= threads) return;
  const int64_t b = i / per_row;
  const int f0 = (int)(i - b * per_row) * VW, left = p.F - f0;
  const S* x = static_cast<const S*>(p.x) + b * p.x_s.batch + f0;
  const S* ig = static_cast<const S*>(p.input_gate) + b * p.input_s.batch + f0;
  const S* dg = static_cast<const S*>(p.decay_gate) + b * p.decay_s.batch + f0;
  const float* carry = p.carry + b * p.F + f0;
  float* final = p.final + b * p.F + f0;
  S* out = static_cast<S*>(p.out) + b * p.F + f0;
  const bool cut = p.done && p.done[b];
  auto step = [&](float xv, float i_, float d, float rate, float h) {
    const Gates g = gates_of<false>(i_, d, rate * LOG2E);
    return apply(cut ? -0.f : g.a, g.wi * xv, h);
  };
  if (left >= VW) {
    Raw<S, VW> rx, ri, rd;
    float h[VW], rate[VW];
    __builtin_memcpy(rx.v, x, sizeof(rx.v));
    __builtin_memcpy(ri.v, ig, sizeof(ri.v));
    __builtin_memcpy(rd.v, dg, sizeof(rd.v));
    __builtin_memcpy(h, carry, sizeof(h));
    __builtin_memcpy(rate, p.rate + f0, sizeof(rate));
#pragma unroll
    for (int k = 0; k < VW; ++k) h[k] = step(widen(rx.v[k]), widen(ri.v[k]), widen(rd.v[k]), rate[k], h[k]);
    store_near<VW>(final, 0, h);
    store_near<VW>(out, 0, h);
  } else {
    for (int k = 0; k < left; ++k) {
      const float h[1] = {step(widen(x[k]), widen(ig[k]), widen(dg[k]), p.rate[f0 + k], carry[k])};
      store_near<1>(final + k, 0, h);
      store_near<1>(out + k, 0, h);
    }
  }
}

// ---- launches
// How a direction lays its lanes: features of a lane and lanes over the
// features, waves, workgroups over the features, segments.
struct Plan {
  int vw, lf, waves, blocks, tile, segment, segments;
};
constexpr int TARGET = 512, FILL = 192;   // workgroups that fill the chip, and most of it
constexpr int SHORT_GROUPS = 4096;        // most workgroups of a launch over short sequences

Plan plan_of(int dtype, bool backward, int batch, int steps, int F) {
  Plan s;
  const int N = backward ? BWD_STEPS : FWD_STEPS;
  s.vw = LANE;
  if (F < s.vw) s.vw = 1;
  // lanes for the features that are there (2048 x 500 steps of 16 bf16 features, both
  // passes: 154 us, 64 lanes 584); where those and the sequences do not fill the chip,
  // fewer side by side, down to a cache line, if that fills most of it (a segment more
  // reads operands twice: 24 x 4093 steps of 640 features 413 us, in segments 491; 24
  // of 256, which it does not fill, 202 in segments, 352 without)
  s.lf = 64;
  const auto groups_at = [&](int lf) { return (int64_t)batch * ceil_div(F, lf * s.vw); };
  const auto fits = [&](int lf) { return 64 / lf * N < 2 * (int64_t)steps; };
  while (s.lf > 8 && s.lf / 2 * s.vw >= F && fits(s.lf / 2)) s.lf /= 2;
  const int line = std::min(s.lf, 128 / (s.vw * (dtype == GATE_F32 ? 4 : 2)));
  if (groups_at(line) >= FILL)
    while (s.lf > line && groups_at(s.lf) < TARGET && fits(s.lf / 2)) s.lf /= 2;
  if (s.vw == 1) s.lf = 8;
  const int slots = 64 / s.lf;
  s.waves = std::min(MAX_WAVES, ceil_div(steps, slots * N));
  s.blocks = ceil_div(F, s.lf * s.vw);
  s.tile = s.waves * slots * N;
  // segments of at least two tiles, as many as fill the chip
  const int64_t groups = (int64_t)batch * s.blocks;
  const int64_t most = std::min<int64_t>(MAX_SEGMENTS, std::max(1, steps / (2 * s.tile)));
  s.segments = groups >= FILL ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(most, TARGET / groups));
  const int tiles = ceil_div(steps, s.tile);
  const int each = ceil_div(tiles, s.segments);
  s.segment = each * s.tile;
  s.segments = ceil_div(tiles, each);
  return s;
}

// The steps between states that the forward leaves: the backward's tile, as a
// power of two.
int save_log2_of(const Plan& bwd) {
  int log2 = 0;
  while ((1 << log2) < bwd.tile) ++log2;
  return log2;
}

int check(const char* what, int dtype, int batch, int steps, int features) {
  if (dtype != GATE_F32 && dtype != GATE_BF16) return set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || features < 0)
    return set_error(PPO_ERR_ARG, "%s: bad size (batch %d steps %d features %d)", what, batch, steps, features);
  if (batch > 1 << 21 || steps > 1 << 30 || features > 1 << 20 || (int64_t)batch * features > 1 << 29)
    return set_error(PPO_ERR_ARG, "%s: batch %d above 2^21, steps %d above 2^30, features %d above 2^20 or batch x "
                     "features above 2^29", what, batch, steps, features);
  return PPO_OK;
}
int check_strides(const char* what, const int64_t* strides, int tensors, int steps) {
  for (int i = 0; i < tensors; ++i)
    if (strides[2 * i + 1] < 0 || (steps > 1 && strides[2 * i + 1] > MAX_STRIDE))
      return set_error(PPO_ERR_ARG, "%s: a step stride of %lld is not from 0 to 2^23", what, (long long)strides[2 * i + 1]);
  return PPO_OK;
}

template <typename S, int VW, int LF, bool BWD>
void launch_shape(hipStream_t st, const GatedArgs& a, const Plan& s, int batch) {
  const unsigned groups = (unsigned)batch * (unsigned)s.blocks;
  const dim3 t(64 * s.waves);
  if (s.segments > 1)
    hipLaunchKernelGGL((gated_maps_kernel<S, VW, LF, BWD>), dim3(groups, s.segments - 1), t, 0, st, a);
  if constexpr (BWD) hipLaunchKernelGGL((gated_bwd_kernel<S, VW, LF>), dim3(groups, s.segments), t, 0, st, a);
  else hipLaunchKernelGGL((gated_fwd_kernel<S, VW, LF>), dim3(groups, s.segments), t, 0, st, a);
}
template <typename S, bool BWD> void launch(hipStream_t st, GatedArgs a, const Plan& s, int batch) {
  constexpr int VW = LANE;
  a.blocks = s.blocks;
  a.segment = s.segment;
  a.segments = s.segments;
  if (s.vw == 1) launch_shape<S, 1, 8, BWD>(st, a, s, batch);
  else if (s.lf == 64) launch_shape<S, VW, 64, BWD>(st, a, s, batch);
  else if (s.lf == 32) launch_shape<S, VW, 32, BWD>(st, a, s, batch);
  else if (s.lf == 16) launch_shape<S, VW, 16, BWD>(st, a, s, batch);
  else launch_shape<S, VW, 8, BWD>(st, a, s, batch);
}

// Short sequences (up to SHORT steps): lanes over the features, workgroups over those
// and the sequences.
struct ShortPlan {
  int vw, lanes_log2;
  unsigned blocks, groups;
};
ShortPlan short_plan_of(bool backward, int batch, int steps, int F) {
  ShortPlan s;
  // (backward, four features of four steps take 256 registers)
  s.vw = F < 4 ? 1 : steps <= 2 ? 4 : steps <= 4 || !backward ? 2 : 1;
  s.lanes_log2 = 0;
  while (s.lanes_log2 < 8 && (s.vw << s.lanes_log2) < F) ++s.lanes_log2;
  s.blocks = (unsigned)ceil_div(F, s.vw << s.lanes_log2);
  s.groups = (unsigned)std::min<int64_t>(ceil_div64(batch, SHORT_THREADS >> s.lanes_log2),
                                         std::max<int64_t>(1, SHORT_GROUPS / s.blocks));
  return s;
}
template <typename S, int VW, int N, bool BWD>
void launch_short_steps(hipStream_t st, const GatedArgs& a, const ShortPlan& s, int batch) {
  const dim3 grid(s.blocks, s.groups), block(SHORT_THREADS);
  if constexpr (BWD) hipLaunchKernelGGL((gated_short_bwd_kernel<S, VW, N>), grid, block, 0, st, a, batch, s.lanes_log2);
  else hipLaunchKernelGGL((gated_short_fwd_kernel<S, VW, N>), grid, block, 0, st, a, batch, s.lanes_log2);
}
template <typename S, int VW, bool BWD>
void launch_short_width(hipStream_t st, const GatedArgs& a, const ShortPlan& s, int batch) {
  if constexpr (VW != 2) {
    if (a.steps == 1) return launch_short_steps<S, VW, 1, BWD>(st, a, s, batch);
    if (a.steps == 2) return launch_short_steps<S, VW, 2, BWD>(st, a, s, batch);
  }
  if constexpr (VW != 4) {
    if (a.steps <= 4) return launch_short_steps<S, VW, 4, BWD>(st, a, s, batch);
  }
  if constexpr (VW == 1 || (VW == 2 && !BWD)) launch_short_steps<S, VW, SHORT, BWD>(st, a, s, batch);
}
template <typename S, bool BWD> void launch_short(hipStream_t st, const GatedArgs& a, int batch) {
  const ShortPlan s = short_plan_of(BWD, batch, a.steps, a.F);
  if (s.vw == 4) launch_short_width<S, 4, BWD>(st, a, s, batch);
  else if (s.vw == 2) launch_short_width<S, 2, BWD>(st, a, s, batch);
  else launch_short_width<S, 1, BWD>(st, a, s, batch);
}

constexpr int RATE_ROWS = 512;   // of partial sums that a workgroup adds

// Rows of a rate's partial sums.
int64_t rate_rows(const Plan& s, int batch, int steps, int F) {
  return steps <= SHORT ? (int64_t)short_plan_of(true, batch, steps, F).groups : (int64_t)batch * s.segments;
}

size_t maps_floats(const Plan& s, int batch, int F) { return s.segments > 1 ? 2 * (size_t)batch * s.segments * F : 0; }

}  // namespace

PPO_EXPORT size_t ppo_gated_scan_workspace(int dtype, int batch, int steps, int features) {
  if (batch <= 0 || steps <= 0 || features <= 0) return 0;
  return sizeof(float) * maps_floats(plan_of(dtype, false, batch, steps, features), batch, features);
}

PPO_EXPORT size_t ppo_gated_scan_states(int dtype, int batch, int steps, int features) {
  if (batch <= 0 || steps <= 0 || features <= 0) return 0;
  const int log2 = save_log2_of(plan_of(dtype, true, batch, steps, features));
  return sizeof(float) * (size_t)batch * ceil_div64(steps, 1ll << log2) * features;
}

PPO_EXPORT int ppo_gated_scan_fwd(void* stream, int dtype, const void* x, const void* input_gate,
                                  const void* decay_gate, const int64_t* strides, const float* rate,
                                  const float* carry, const uint8_t* done, const int32_t* lengths, void* out,
                                  float* final, float* states, void* workspace, size_t workspace_bytes, int batch,
                                  int steps, int features) {
  const char* what = "ppo_gated_scan_fwd";
  if (int rc = check(what, dtype, batch, steps, features)) return rc;
  if (batch == 0 || steps == 0 || features == 0) return PPO_OK;
  if (!x || !input_gate || !decay_gate || !strides || !rate || !out || !final)
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 3, steps)) return rc;
  const size_t need = ppo_gated_scan_workspace(dtype, batch, steps, features);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  GatedArgs a{};
  a.x = x;
  a.input_gate = input_gate;
  a.decay_gate = decay_gate;
  a.rate = rate;
  a.carry = carry;
  a.done = done;
  a.lengths = lengths;
  a.out = out;
  a.final = final;
  a.states = states;
  a.maps = static_cast<float*>(workspace);
  a.x_s = RowStride{strides[0], strides[1]};
  a.input_s = RowStride{strides[2], strides[3]};
  a.decay_s = RowStride{strides[4], strides[5]};
  a.steps = steps;
  a.F = features;
  a.save_log2 = save_log2_of(plan_of(dtype, true, batch, steps, features));
  a.saved = (int)ceil_div64(steps, 1ll << a.save_log2);
  const Plan s = plan_of(dtype, false, batch, steps, features);
  if (steps <= SHORT) {
    if (dtype == GATE_F32) launch_short<float, false>(as_stream(stream), a, batch);
    else launch_short<uint16_t, false>(as_stream(stream), a, batch);
    return check_launch(what);
  }
  if (dtype == GATE_F32) launch<float, false>(as_stream(stream), a, s, batch);
  else launch<uint16_t, false>(as_stream(stream), a, s, batch);
  return check_launch(what);
}

PPO_EXPORT size_t ppo_gated_scan_bwd_workspace(int dtype, int batch, int steps, int features) {
  if (batch <= 0 || steps <= 0 || features <= 0) return 0;
  const Plan s = plan_of(dtype, true, batch, steps, features);
  const int64_t rows = rate_rows(s, batch, steps, features);
  const int64_t sums = rows + (rows > RATE_ROWS ? ceil_div64(rows, RATE_ROWS) : 0);
  return sizeof(float) * (maps_floats(s, batch, features) + (size_t)sums * features);
}

PPO_EXPORT int ppo_gated_scan_bwd(void* stream, int dtype, const void* x, const void* input_gate,
                                  const void* decay_gate, const void* dout, const int64_t* strides, const float* rate,
                                  const uint8_t* done, const int32_t* lengths, const float* states,
                                  const float* dfinal, void* dx, void* dinput_gate, void* ddecay_gate, float* drate,
                                  float* dcarry, void* workspace, size_t workspace_bytes, int batch, int steps,
                                  int features) {
  const char* what = "ppo_gated_scan_bwd";
  if (int rc = check(what, dtype, batch, steps, features)) return rc;
  if (batch == 0 || steps == 0 || features == 0) return PPO_OK;
  if (!x || !input_gate || !decay_gate || !dout || !strides || !rate || !states || !dx || !dinput_gate || !ddecay_gate)
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 4, steps)) return rc;
  const size_t need = ppo_gated_scan_bwd_workspace(dtype, batch, steps, features);
  if (!workspace || workspace_bytes < need)
    return set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  const Plan s = plan_of(dtype, true, batch, steps, features);
  GatedArgs a{};
  a.x = x;
  a.input_gate = input_gate;
  a.decay_gate = decay_gate;
  a.dout = dout;
  a.rate = rate;
  a.done = done;
  a.lengths = lengths;
  a.states = const_cast<float*>(states);
  a.dfinal = dfinal;
  a.dx = dx;
  a.dinput_gate = dinput_gate;
  a.ddecay_gate = ddecay_gate;
  a.dcarry = dcarry;
  a.maps = static_cast<float*>(workspace);
  float* partials = a.maps + maps_floats(s, batch, features);
  a.partials = drate ? partials : nullptr;
  a.x_s = RowStride{strides[0], strides[1]};
  a.input_s = RowStride{strides[2], strides[3]};
  a.decay_s = RowStride{strides[4], strides[5]};
  a.dout_s = RowStride{strides[6], strides[7]};
  a.steps = steps;
  a.F = features;
  a.save_log2 = save_log2_of(s);
  a.saved = (int)ceil_div64(steps, 1ll << a.save_log2);
  if (steps <= SHORT && dtype == GATE_F32) launch_short<float, true>(as_stream(stream), a, batch);
  else if (steps <= SHORT) launch_short<uint16_t, true>(as_stream(stream), a, batch);
  else if (dtype == GATE_F32) launch<float, true>(as_stream(stream), a, s, batch);
  else launch<uint16_t, true>(as_stream(stream), a, s, batch);
  if (drate) {
    const int64_t rows = rate_rows(s, batch, steps, features);
    const unsigned columns = (unsigned)ceil_div(features, 64);
    if (rows > RATE_ROWS) {
      const int64_t some = ceil_div64(rows, RATE_ROWS);
      float* sums = partials + rows * features;
      hipLaunchKernelGGL(gated_rate_kernel, dim3(columns, (unsigned)some), dim3(1024), 0, as_stream(stream), partials, rows,
                         RATE_ROWS, features, sums);
      hipLaunchKernelGGL(gated_rate_kernel, dim3(columns), dim3(1024), 0, as_stream(stream), sums, some, (int)some, features,
                         drate);
    } else {
      hipLaunchKernelGGL(gated_rate_kernel, dim3(columns), dim3(1024), 0, as_stream(stream), partials, rows, (int)rows,
                         features, drate);
    }
  }
  return check_launch(what);
}

PPO_EXPORT int ppo_gated_scan_step(void* stream, int dtype, const void* x, const void* input_gate,
                                   const void* decay_gate, const int64_t* strides, const float* rate,
                                   const float* carry, const uint8_t* done, void* out, float* final, int batch,
                                   int features) {
  const char* what = "ppo_gated_scan_step";
  if (int rc = check(what, dtype, batch, 1, features)) return rc;
  if (batch == 0 || features == 0) return PPO_OK;
  if (!x || !input_gate || !decay_gate || !strides || !rate || !carry || !out || !final)
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  GatedArgs a{};
  a.x = x;
  a.input_gate = input_gate;
  a.decay_gate = decay_gate;
  a.rate = rate;
  a.carry = carry;
  a.done = done;
  a.out = out;
  a.final = final;
  a.x_s = RowStride{strides[0], 0};
  a.input_s = RowStride{strides[1], 0};
  a.decay_s = RowStride{strides[2], 0};
  a.steps = 1;
  a.F = features;
  const int per_row = ceil_div(features, 4);
  const int64_t threads = (int64_t)batch * per_row;
  const dim3 grid((unsigned)ceil_div64(threads, 256)), block(256);
  if (dtype == GATE_F32) hipLaunchKernelGGL((gated_step_kernel<float, 4>), grid, block, 0, as_stream(stream), a, threads, per_row);
  else hipLaunchKernelGGL((gated_step_kernel<uint16_t, 4>), grid, block, 0, as_stream(stream), a, threads, per_row);
  return check_launch(what);
}
