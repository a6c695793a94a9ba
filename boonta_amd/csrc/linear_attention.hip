// Linear attention with a decay for each head: the recurrence of a recurrent
// torso whose state is a matrix, in chunks of steps (training minibatches,
// prompts) with its vector-Jacobian product, and one step of it (rollouts).
//
// Per sequence b and head h, lam = exp(log_decay[h]), n = lengths[b] steps:
//   S_t = lam (done_t ? 0 : S_{t-1}) + k_t v_t^T   (S_{-1} = carry)
//   o_t = scale q_t S_t                            (o_t = 0 for t >= n)
// and with D_t the cotangent of S_t:
//   D_t  = scale q_t do_t^T + (done_{t+1} ? 0 : lam D_{t+1}),  D_{n-1} += dfinal
//   dq_t = scale do_t S_t^T,  dk_t = v_t D_t^T,  dv_t = k_t D_t
//   dcarry = done_0 ? 0 : lam D_0
//
// All four sequences of outputs are one contraction in one of two directions:
//   out_r = x_r St_r,  St_r = lam St_{r-1} + y_r z_r^T
//   o:  x, y, z = q, k, v forward      dq: do, v, k forward (St = S^T)
//   dv: k, q, do backward (St = D)     dk: v, do, q backward (St = D^T)
// so one kernel computes each, and the three of the backward pass run side by
// side in one launch.  In a chunk of C steps entered with state St:
//   out_i = lam^{i+1} x_i St + sum_{j <= i} lam^{i-j} (x_i . y_j) z_j
//   St'   = lam^n St + sum_j y_j (lam^{n-1-j} z_j)^T
// where a reset between two steps removes their term (a 64-bit mask of the
// chunk's resets gives the last reset before each step), and every power's
// exponent is >= 0, so nothing grows for lam <= 1.
#include "split_f32.h"

#include <algorithm>

namespace {

using ppo::pack_bf16;

enum AttnDtype { ATTN_F32 = 0, ATTN_BF16 = 1 };

// [batch, steps, heads, width] operand, element strides; `group` heads of the
// problem share one of the operand's.
struct Operand {
  const void* p;
  int64_t sb, st, sh;
  int group, width;
};

struct Contraction {
  Operand x, y, z;
  void* out;              // [batch, steps, heads, z.width]
  const float* carry;     // [batch * heads, K V] state before the first step, or null (zeros)
  float* states;          // [batch * heads, segments - 1, K V]: states entering the segments after the first
  float* final;           // [batch * heads, K V] state after the last step, or null
  int transposed;         // St is the transpose of the K V matrix in memory
  int backward;           // steps from the last to the first
  int wide;               // out holds float32 (summed over heads that share an operand), not the operands' type
  float intra, inter, update;  // factors of the pair sum, of x St, and of y z^T in St
};

struct AttnArgs {
  Contraction role[3];
  const float* log_decay;   // [heads]
  const uint8_t* done;      // [batch, steps], or null
  const int32_t* lengths;   // [batch], or null
  float* factors;           // [batch * heads, segments - 1]: a segment's decay of its entry state (-1: reset)
  int steps, heads, segments, seg_steps, roles;
};

// ---- per type: chunks of 128 bytes of steps; a lane's MFMA operand of 16
// bytes (FR values).  One contraction block is 4 FR deep: a 16x16x32 bf16
// MFMA, or four 16x16x4 fp32 MFMAs, whose lane group g supplies values
// 4g .. 4g+3 of each 16 rows, which is how the accumulators hold them: a
// state tile is an operand without a move.
template <typename T> struct Type;

template <> struct Type<uint16_t> {
  typedef bf16x8 Frag;
  static constexpr int FR = 8, C = 64, PIECES = 3;
  static __device__ __forceinline__ floatx4 mma(Frag a, Frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Type<float> {
  typedef floatx4 Frag;
  static constexpr int FR = 4, C = 32, PIECES = 1;
  static __device__ __forceinline__ floatx4 mma(Frag a, Frag b, floatx4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ bf16x8 join(floatx4 lo, floatx4 hi) {
  uint4 w;
  w.x = pack_bf16(lo[0], lo[1]);
  w.y = pack_bf16(lo[2], lo[3]);
  w.z = pack_bf16(hi[0], hi[1]);
  w.w = pack_bf16(hi[2], hi[3]);
  return __builtin_bit_cast(bf16x8, w);
}

// The state as an operand over its rows: contraction block kb of n-tile nt.
// bf16: the state itself stays float32; what enters the product is rounded
// once, an error of the size of the output's own rounding.
template <int RT> __device__ __forceinline__ bf16x8 state_frag(const floatx4 (&s)[RT][2], int kb, int nt, uint16_t) {
  return join(s[2 * kb][nt], s[2 * kb + 1][nt]);
}
template <int RT> __device__ __forceinline__ floatx4 state_frag(const floatx4 (&s)[RT][2], int kb, int nt, float) {
  return s[kb][nt];
}

// z times its steps' weights, as operands whose sum is the product to float32:
// one float32, or three bf16 pieces, each what the ones before leave (the
// states are float32 sums of exact products of these).
__device__ __forceinline__ void weigh(bf16x8 z, const float (&w)[8], bf16x8 (&p)[3]) {
  const uint4 u = __builtin_bit_cast(uint4, z);
  const uint32_t q[4] = {u.x, u.y, u.z, u.w};
  floatx4 lo, hi;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lo[2 * i] = __uint_as_float(q[i] << 16) * w[2 * i];
    lo[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u) * w[2 * i + 1];
    hi[2 * i] = __uint_as_float(q[2 + i] << 16) * w[4 + 2 * i];
    hi[2 * i + 1] = __uint_as_float(q[2 + i] & 0xffff0000u) * w[5 + 2 * i];
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = ppo::split_piece(lo, hi);
}
__device__ __forceinline__ void weigh(floatx4 z, const float (&w)[4], floatx4 (&p)[1]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) p[0][e] = z[e] * w[e];
}

// XOR of the 16-byte chunk index (0 .. 7) of row r in a tile of 128-byte rows:
// 16 consecutive rows read at one chunk, and 8-byte writes to one chunk of
// rows 8 apart, fall on different banks.
__device__ __forceinline__ int swizzle(int r) { return ((r >> 1) ^ (r >> 3)) & 7; }

// Byte of an operand (row 16 tile + l16, chunk 4 tb + g4) in such a tile, from
// the lane's own byte of tile 0, chunk 0: the swizzle of row 16 tile + l16 is
// that of l16 with 2 (tile & 3) in it.
__device__ __forceinline__ int tile_byte(int lane_byte, int tile, int tb) {
  return (lane_byte ^ (((4 * tb) ^ (2 * (tile & 3))) << 4)) + tile * 2048;
}

struct Regs {
  uint4 v[4];
};

// 16 bytes of a row, elements c0 .. c0 + FR - 1, as loaded and then (once they
// are there: a use would wait for them) with what is past the row's `width`
// zeros.  No branch on the lane: the last chunk of a width that FR does not
// divide is read from its end and shifted.  Rows need no alignment beyond
// their elements'.
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const char* row, uint32_t byte, int c0, int width) {
  constexpr int FR = Type<T>::FR;
  uint4 v;
  if (width >= FR) {
    __builtin_memcpy(&v, row + byte, 16);
  } else {
    T e[FR];
#pragma unroll
    for (int j = 0; j < FR; ++j) {
      T x;
      __builtin_memcpy(&x, row + byte + min(j, width - 1) * sizeof(T), sizeof(T));
      e[j] = c0 + j < width ? x : T(0);
    }
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}
// The column a chunk's load starts at.
template <typename T> __device__ __forceinline__ int load_column(int c0, int width) {
  return width >= Type<T>::FR ? min(c0, width - Type<T>::FR) : 0;
}
template <typename T>
__device__ __forceinline__ uint4 trim_chunk(uint4 v, int c0, int width) {
  constexpr int FR = Type<T>::FR;
  if (width < FR) return v;
  const int over = c0 + FR - width;   // elements past the row
  if (over <= 0) return v;
  const int s = min(over, FR) * (int)sizeof(T) * 8;
  const uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
  const uint64_t l = s < 64 ? lo >> s | hi << (64 - s) : s < 128 ? hi >> (s - 64) : 0;
  const uint64_t h = s < 64 ? hi >> s : 0;
  return make_uint4((uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32));
}

__device__ __forceinline__ bool odd_exponent(uint4 v, uint16_t) {  // an infinity or NaN among eight bf16
  auto f = [](uint32_t u) { return (u & 0x7f807f80u) + 0x00800080u; };
  return ((f(v.x) | f(v.y) | f(v.z) | f(v.w)) & 0x80008000u) != 0;
}
__device__ __forceinline__ bool odd_exponent(uint4 v, float) {
  auto f = [](uint32_t u) { return (u & 0x7f800000u) + 0x00800000u; };
  return ((f(v.x) | f(v.y) | f(v.z) | f(v.w)) & 0x80000000u) != 0;
}

// Four rows' chunks of one step each as columns: element j of the chunk, over
// the four steps.
__device__ __forceinline__ void write_transposed(char* t, int dim0, int tg, const Regs& r, uint16_t) {
  const uint32_t* a = reinterpret_cast<const uint32_t*>(&r.v[0]);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(&r.v[1]);
  const uint32_t* c = reinterpret_cast<const uint32_t*>(&r.v[2]);
  const uint32_t* d = reinterpret_cast<const uint32_t*>(&r.v[3]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = dim0 + j, w = j >> 1;
    uint2 x;
    // bytes of two words by v_perm: the low or high half of each
    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
    x.x = __builtin_amdgcn_perm(b[w], a[w], sel);
    x.y = __builtin_amdgcn_perm(d[w], c[w], sel);
    *reinterpret_cast<uint2*>(t + row * 128 + (((tg >> 1) ^ swizzle(row)) << 4) + ((tg & 1) << 3)) = x;
  }
}
__device__ __forceinline__ void write_transposed(char* t, int dim0, int tg, const Regs& r, float) {
  const uint32_t* a = reinterpret_cast<const uint32_t*>(&r.v[0]);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(&r.v[1]);
  const uint32_t* c = reinterpret_cast<const uint32_t*>(&r.v[2]);
  const uint32_t* d = reinterpret_cast<const uint32_t*>(&r.v[3]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = dim0 + j;
    *reinterpret_cast<uint4*>(t + row * 128 + ((tg ^ swizzle(row)) << 4)) = make_uint4(a[j], b[j], c[j], d[j]);
  }
}

// Row-major rows; bf16 columns 16 h + 4 g + j of each 32 at 8 g + 4 h + j, so
// that a lane's operand (see Type) is 16 contiguous bytes.
__device__ __forceinline__ void write_rows(char* t, int pitch, int dc, int tg, const Regs& r, uint16_t) {
  const int h = (dc & 3) >> 1, g = 2 * (dc & 1);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    char* p = t + (4 * tg + e) * pitch + 64 * (dc >> 2) + 16 * g + 8 * h;
    *reinterpret_cast<uint2*>(p) = make_uint2(r.v[e].x, r.v[e].y);
    *reinterpret_cast<uint2*>(p + 16) = make_uint2(r.v[e].z, r.v[e].w);
  }
}
__device__ __forceinline__ void write_rows(char* t, int pitch, int dc, int tg, const Regs& r, float) {
#pragma unroll
  for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(t + (4 * tg + e) * pitch + 16 * dc) = r.v[e];
}
__device__ __forceinline__ float row_value(const char* t, int pitch, int i, int c, uint16_t) {
  const int at = (c & ~31) + 8 * ((c >> 2) & 3) + 4 * ((c >> 4) & 1) + (c & 3);
  return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(t + i * pitch)[at] << 16);
}
__device__ __forceinline__ float row_value(const char* t, int pitch, int i, int c, float) {
  return reinterpret_cast<const float*>(t + i * pitch)[c];
}
__device__ __forceinline__ float column_value(const char* t, int row, int i, uint16_t) {
  const char* p = t + row * 128 + (((i >> 3) ^ swizzle(row)) << 4);
  return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i & 7] << 16);
}
__device__ __forceinline__ float column_value(const char* t, int row, int i, float) {
  return reinterpret_cast<const float*>(t + row * 128 + (((i >> 2) ^ swizzle(row)) << 4))[i & 3];
}

// Four consecutive outputs of a row, `left` of them inside it.
__device__ __forceinline__ void store4(uint16_t* p, floatx4 v, int left) {
  uint2 w;
  w.x = pack_bf16(v[0], v[1]);
  w.y = pack_bf16(v[2], v[3]);
  if (left >= 4) {
    __builtin_memcpy(p, &w, 8);
  } else {
    if (left > 0) p[0] = (uint16_t)w.x;
    if (left > 1) p[1] = (uint16_t)(w.x >> 16);
    if (left > 2) p[2] = (uint16_t)w.y;
  }
}
__device__ __forceinline__ void store4(float* p, floatx4 v, int left) {
  if (left >= 4) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) p[e] = v[e];
  }
}

// The value, as if computed here: what depends on it is not moved out of the
// loop, where it would hold registers for a part that is seldom run.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float power(float g2, int e) { return __builtin_amdgcn_exp2f(g2 * (float)e); }

// One workgroup per (role, head, segment, sequence): D / 32 waves, each with
// 32 columns of the D x D state in its accumulators.  Widths below D are
// padded with zeros.  Each chunk of x, y, z is loaded once, a chunk ahead, into
// registers, and laid out in LDS by rows (x, y: the pair products) and by
// columns (y, z: contractions over steps).  STATE: only the state, from zeros,
// for the segments before the last.
template <typename T, int D, bool STATE>
__global__ void __launch_bounds__(2 * D, 2) attention_kernel(AttnArgs p) {
  typedef typename Type<T>::Frag Frag;
  constexpr int FR = Type<T>::FR, C = Type<T>::C, W = D / 32, KB = D / (4 * FR), RT = D / 16, QT = C / 16;
  constexpr int PITCH = D * (int)sizeof(T) + 16, ROWS = C * PITCH, COLS = D * 128;
  __shared__ __attribute__((aligned(16))) char smem[(STATE ? 0 : 2 * ROWS + C * 128) + 2 * COLS + 16];
  char* const yt = smem;
  char* const zt = smem + COLS;
  char* const xr = STATE ? nullptr : smem + 2 * COLS;
  char* const yr = STATE ? nullptr : smem + 2 * COLS + ROWS;
  char* const pr = STATE ? nullptr : smem + 2 * COLS + 2 * ROWS;
  volatile int* const odd = reinterpret_cast<volatile int*>(smem + sizeof(smem) - 16);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g4 = lane >> 4;
  int at = ppo::xcd_tile().n;
  const int role = at % p.roles;
  at /= p.roles;
  const int head = at % p.heads;
  at /= p.heads;
  const int segs = STATE ? p.segments - 1 : p.segments;
  const int seg = at % segs;
  const int b = at / segs;
  const Contraction& c = p.role[role];
  const int64_t bh = (int64_t)b * p.heads + head;
  const int R = c.x.width, N = c.z.width;
  const int64_t KV = (int64_t)R * N;
  const bool back = c.backward;

  const int len = p.lengths ? min(max(p.lengths[b], 0), p.steps) : p.steps;
  float g2 = p.log_decay[head] * 1.44269504088896341f;
  g2 = g2 < -1e30f ? -1e30f : g2;  // (a decay of zero: 0 times an infinite exponent is no number)
  const uint8_t* done = p.done ? p.done + (int64_t)b * p.steps : nullptr;
  const int first = seg * p.seg_steps;                                        // steps in the order of processing
  const int last = min(len, first + p.seg_steps);

  const T* xp = static_cast<const T*>(c.x.p) + b * c.x.sb + (head / c.x.group) * c.x.sh;
  const T* yp = static_cast<const T*>(c.y.p) + b * c.y.sb + (head / c.y.group) * c.y.sh;
  const T* zp = static_cast<const T*>(c.z.p) + b * c.z.sb + (head / c.z.group) * c.z.sh;
  const int64_t pitch_o = (int64_t)p.heads * N, base_o = ((int64_t)b * p.steps * p.heads + head) * N;

  // rows past the sequence's end hold zeros
  if constexpr (!STATE) {
    const int end = min(p.steps, first + p.seg_steps);
    for (int t = max(len, first) + wave; t < end; t += W)
      for (int n = lane; n < N; n += 64) {
        if (c.wide) static_cast<float*>(c.out)[base_o + t * pitch_o + n] = 0.f;
        else static_cast<T*>(c.out)[base_o + t * pitch_o + n] = T(0);
      }
  }

  // the state entering the segment: rows 16 rt + 4 g4 + e, columns 32 wave + 16 nt + l16
  floatx4 S[RT][2];
  const float* entry = nullptr;
  if constexpr (!STATE) entry = seg == 0 ? (c.carry ? c.carry + bh * KV : nullptr)
                                         : c.states + (bh * (p.segments - 1) + seg - 1) * KV;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * rt + 4 * g4 + e, n = 32 * wave + 16 * nt + l16;
        S[rt][nt][e] = 0.f;
        if (entry && r < R && n < N) S[rt][nt][e] = entry[c.transposed ? (int64_t)n * R + r : (int64_t)r * N + n];
      }

  // this thread's share of a chunk: steps 4 tg .. 4 tg + 3, columns FR dc ..
  const int dc = tid % (D / FR), tg = tid / (D / FR);
  Regs rx, ry, rz;
  auto fetch = [&](Regs& r, const Operand& o, const T* base, int r0) {
    const int st = (int)o.st, col = load_column<T>(dc * FR, o.width);
    if (r0 + C <= last) {  // a whole chunk: rows at one offset a lane from uniform addresses
      const T* low = base + (int64_t)(back ? len - r0 - C : r0) * st;
      const uint32_t byte = (uint32_t)((back ? C - 4 - 4 * tg : 4 * tg) * st + col) * (uint32_t)sizeof(T);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r.v[e] = load_chunk<T>(reinterpret_cast<const char*>(low + (back ? 3 - e : e) * st), byte, dc * FR, o.width);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = min(4 * tg + e, last - 1 - r0);
        const T* low = base + (int64_t)(back ? len - last : r0) * st;
        const uint32_t byte = (uint32_t)((back ? last - 1 - r0 - s : s) * st + col) * (uint32_t)sizeof(T);
        r.v[e] = load_chunk<T>(reinterpret_cast<const char*>(low), byte, dc * FR, o.width);
      }
    }
  };
  auto finish = [&](Regs& r, int width, int n) {
    if (width < D) {
      const int c0 = here(dc * FR);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.v[e] = trim_chunk<T>(r.v[e], c0, width);
    }
    if (n < C) {
      const int s = here(4 * tg);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s + e >= n) r.v[e] = make_uint4(0, 0, 0, 0);
    }
  };
  auto fetch_done = [&](int r0) -> int {  // whether the state entering step r0 + lane is dropped
    const int s = r0 + lane;
    if (!done || lane >= C || s >= last) return 0;
    if (!back) return done[s];
    return s > 0 ? done[len - s] : 0;
  };
  int cut_next = 0;
  if (first < last) {
    if constexpr (!STATE) fetch(rx, c.x, xp, first);
    fetch(ry, c.y, yp, first);
    fetch(rz, c.z, zp, first);
    cut_next = fetch_done(first);
  }
  if (tid < 4) odd[tid] = 0;
  if constexpr (!STATE)
    for (int i = tid; i < C * 8; i += 2 * D) reinterpret_cast<uint4*>(pr)[i] = make_uint4(0, 0, 0, 0);
  lds_barrier();

  const int lane_byte = l16 * 128 + ((g4 ^ swizzle(l16)) << 4);
  float whole = 1.f;  // the segment's decay of its entry state, -1 once a reset dropped it
  for (int r0 = first, it = 0; r0 < last; r0 += C, ++it) {
    const int n = min(C, last - r0);
    const uint64_t cut = __ballot(cut_next != 0);
    if constexpr (!STATE) finish(rx, R, n);
    finish(ry, R, n);
    finish(rz, N, n);
    bool is_odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) is_odd |= odd_exponent(ry.v[e], T()) | odd_exponent(rz.v[e], T());
    if (__ballot(is_odd) && lane == 0) odd[it & 1] = 1;
    if constexpr (!STATE) {
      write_rows(xr, PITCH, dc, tg, rx, T());
      write_rows(yr, PITCH, dc, tg, ry, T());
    }
    write_transposed(yt, dc * FR, tg, ry, T());
    write_transposed(zt, dc * FR, tg, rz, T());
    if (r0 + C < last) {
      if constexpr (!STATE) fetch(rx, c.x, xp, r0 + C);
      fetch(ry, c.y, yp, r0 + C);
      fetch(rz, c.z, zp, r0 + C);
      cut_next = fetch_done(r0 + C);
    }
    lds_barrier();
    const bool careful = __builtin_amdgcn_readfirstlane(odd[it & 1]);
    if (tid == 0) odd[(it + 1) & 1] = 0;
    // a backward sequence's first step takes the state as it is
    const int skip = back && r0 == 0 ? 1 : 0;
    const int last_cut = cut ? 63 - __clzll(cut) : -1;  // the last reset of the chunk
    const float fade = power(g2, n - skip);

    if (__builtin_expect(careful, 0)) {
      // An infinity or NaN in y or z: the products above multiply it by the
      // zeros of masked pairs, so the chunk is stepped through as defined.
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int g4 = here(lane >> 4), l16 = here(lane & 15);
        const float f = power(g2, i == 0 && skip ? 0 : 1);
        const bool drop = cut >> i & 1;
        float o[2] = {0.f, 0.f};
        const int col0 = 32 * wave + l16;
        const float z0 = column_value(zt, col0, i, T()) * c.update, z1 = column_value(zt, col0 + 16, i, T()) * c.update;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 16 * rt + 4 * g4 + e;
            const float y = column_value(yt, r, i, T());
            const bool in = r < R;
            S[rt][0][e] = in ? __fmaf_rn(y, z0, drop ? 0.f : f * S[rt][0][e]) : 0.f;
            S[rt][1][e] = in ? __fmaf_rn(y, z1, drop ? 0.f : f * S[rt][1][e]) : 0.f;
            if constexpr (!STATE) {
              const float x = row_value(xr, PITCH, i, r, T());
              if (in) {
                o[0] = __fmaf_rn(x, S[rt][0][e], o[0]);
                o[1] = __fmaf_rn(x, S[rt][1][e], o[1]);
              }
            }
          }
        if constexpr (!STATE) {
          const int64_t row = base_o + (int64_t)(back ? len - 1 - (r0 + i) : r0 + i) * pitch_o;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const float v = ppo::add_xor32(ppo::add_xor16(o[nt])) * c.inter;
            const int col = col0 + 16 * nt;
            if (g4 == 0 && col < N) {
              if (c.wide) static_cast<float*>(c.out)[row + col] = v;
              else store4(static_cast<T*>(c.out) + row + col, floatx4{v, v, v, v}, 1);
            }
          }
        }
      }
      lds_barrier();
      if constexpr (!STATE) {
        lds_barrier();
      }
    } else {
      floatx4 acc[2][QT];
      if constexpr (!STATE) {
        // pair products, keys as rows so that a lane holds four keys of one
        // query: tile (qt, kt) of the lower triangle, dealt to the waves
#pragma unroll 1
        for (int idx = wave; idx < QT * (QT + 1) / 2; idx += W) {
          const int qt = QT == 2 ? (idx > 0) : (idx > 0) + (idx > 2) + (idx > 5);
          const int kt = idx - qt * (qt + 1) / 2;
          floatx4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const Frag ya = *reinterpret_cast<const Frag*>(yr + (16 * kt + l16) * PITCH + 64 * kb + 16 * g4);
            const Frag xb = *reinterpret_cast<const Frag*>(xr + (16 * qt + l16) * PITCH + 64 * kb + 16 * g4);
            a = Type<T>::mma(ya, xb, a);
          }
          const int i = 16 * qt + l16, j0 = 16 * kt + 4 * g4;
          const uint64_t upto = cut & (~0ull >> (63 - i));
          const int from = upto ? 63 - __clzll(upto) : 0;  // the last reset up to step i
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + e;
            a[e] = j <= i && j >= from ? a[e] * (c.intra * power(g2, i - j)) : 0.f;
          }
          if constexpr (sizeof(T) == 2) {
            const int chunk = 2 * kt + (g4 >> 1);
            *reinterpret_cast<uint2*>(pr + i * 128 + ((chunk ^ swizzle(i)) << 4) + ((g4 & 1) << 3)) =
                make_uint2(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]));
          } else {
            *reinterpret_cast<floatx4*>(pr + i * 128 + (((4 * kt + g4) ^ swizzle(i)) << 4)) = a;
          }
        }
        // x times the entry state (rows: its columns)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) acc[nt][qt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const Frag s0 = state_frag(S, kb, 0, T()), s1 = state_frag(S, kb, 1, T());
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const Frag xb = *reinterpret_cast<const Frag*>(xr + (16 * qt + l16) * PITCH + 64 * kb + 16 * g4);
            acc[0][qt] = Type<T>::mma(s0, xb, acc[0][qt]);
            acc[1][qt] = Type<T>::mma(s1, xb, acc[1][qt]);
          }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const int i = 16 * qt + l16;
          const bool reach = (cut & (~0ull >> (63 - i))) == 0;
          const float f = c.inter * power(g2, i + 1 - skip);
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][qt][e] = reach ? acc[nt][qt][e] * f : 0.f;
        }
        lds_barrier();
      }
      if constexpr (!STATE) {
        // the pair products times z, and the outputs
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
          Frag z[2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
            z[nt] = *reinterpret_cast<const Frag*>(zt + tile_byte(lane_byte, 2 * wave + nt, tb));
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            if (16 * qt + 15 < 4 * FR * tb) continue;  // keys after the queries
            const Frag pb = *reinterpret_cast<const Frag*>(pr + tile_byte(lane_byte, qt, tb));
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) acc[nt][qt] = Type<T>::mma(z[nt], pb, acc[nt][qt]);
          }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const int i = 16 * qt + l16;
          if (i < n) {
            const int64_t row = base_o + (int64_t)(back ? len - 1 - (r0 + i) : r0 + i) * pitch_o;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const int col = 32 * wave + 16 * nt + 4 * g4;
              if (c.wide) store4(static_cast<float*>(c.out) + row + col, acc[nt][qt], N - col);
              else store4(static_cast<T*>(c.out) + row + col, acc[nt][qt], N - col);
            }
          }
        }
      }
      // state: its rows by y's columns, contracted over the steps
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[rt][nt][e] = cut ? 0.f : S[rt][nt][e] * fade;
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        Frag w[2][Type<T>::PIECES];
        float weight[FR];
#pragma unroll
        for (int e = 0; e < FR; ++e) {
          const int j = 4 * FR * tb + FR * g4 + e;
          weight[e] = j < n && j >= last_cut ? c.update * power(g2, n - 1 - j) : 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          weigh(*reinterpret_cast<const Frag*>(zt + tile_byte(lane_byte, 2 * wave + nt, tb)), weight, w[nt]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const Frag ya = *reinterpret_cast<const Frag*>(yt + tile_byte(lane_byte, rt, tb));
#pragma unroll
          for (int q = Type<T>::PIECES - 1; q >= 0; --q)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) S[rt][nt] = Type<T>::mma(ya, w[nt][q], S[rt][nt]);
        }
      }
      lds_barrier();
    }
    whole = cut || whole < 0.f ? -1.f : whole * fade;
  }

  float* exit = STATE ? c.states + (bh * (p.segments - 1) + seg) * KV
                      : (c.final && seg == p.segments - 1 ? c.final + bh * KV : nullptr);
  if (!exit) return;
  if (STATE && tid == 0) p.factors[bh * (p.segments - 1) + seg] = whole;
  // the cotangent of the state before the first step
  float f = 1.f;
  bool drop = false;
  if (!STATE && back && len > 0) {
    f = power(g2, 1);
    drop = done && done[0];
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * rt + 4 * g4 + e, n = 32 * wave + 16 * nt + l16;
        if (r < R && n < N)
          exit[c.transposed ? (int64_t)n * R + r : (int64_t)r * N + n] = drop ? 0.f : S[rt][nt][e] * f;
      }
}

// The states entering each segment after the first, from what each segment
// before the last adds from zeros and how it fades what enters it; in place.
__global__ void __launch_bounds__(256) join_segments_kernel(float* states, const float* factors, const float* carry,
                                                            int64_t KV, int segs) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, bh = blockIdx.y;
  if (i >= KV) return;
  float s = carry ? carry[bh * KV + i] : 0.f;
  float* p = states + bh * segs * KV + i;
  const float* f = factors + bh * segs;
  for (int k0 = 0; k0 < segs; k0 += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = p[min(k0 + k, segs - 1) * KV];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k0 + k < segs) {
        const float fade = f[k0 + k];
        s = fade < 0.f ? v[k] : __fmaf_rn(fade, s, v[k]);
        p[(k0 + k) * KV] = s;
      }
  }
}

// Gradients of heads that `group` query heads share: their sum.
template <typename T>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* x, T* out, int64_t n, int width, int group) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float* p = x + i / width * width * group + i % width;
  float s = 0.f;
  for (int j = 0; j < group; ++j) s += p[(int64_t)j * width];
  store4(out + i, floatx4{s, s, s, s}, 1);
}

// ---- one step
struct StepArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t qb, qh, kb, kh, vb, vh;
  const float* log_decay;
  const uint8_t* done;
  const float* state;
  float* state_out;
  void* out;
  float scale;
  int heads, group, K, V, slices, slice;
};

__device__ __forceinline__ float value(const uint16_t* p, int64_t i) { return __uint_as_float((uint32_t)p[i] << 16); }
__device__ __forceinline__ float value(const float* p, int64_t i) { return p[i]; }

// A workgroup holds a slice of one head's columns: VEC columns a lane, CL
// lanes across, the rest down the rows, RB rows a lane in flight.  The state
// is read and written once; bound by HBM.
template <typename T, int VEC, int CL>
__global__ void __launch_bounds__(256) attention_step_kernel(StepArgs a) {
  constexpr int RL = 256 / CL, RB = 8;
  __shared__ float sq[128], sk[128];
  __shared__ float part[4][CL * VEC];
  const int tid = threadIdx.x, cl = tid % CL, rl = tid / CL;
  const int slice = blockIdx.x % a.slices;
  const int64_t bh = blockIdx.x / a.slices;
  const int head = (int)(bh % a.heads);
  const int64_t b = bh / a.heads;
  const int n0 = slice * a.slice + cl * VEC;
  const bool ok = cl * VEC < a.slice && n0 < a.V;
  const int64_t base = bh * a.K * a.V + n0;
  const bool cut = a.done && a.done[b];
  for (int r = tid; r < a.K; r += 256) {
    sq[r] = value(static_cast<const T*>(a.q), b * a.qb + head * a.qh + r);
    sk[r] = value(static_cast<const T*>(a.k), b * a.kb + (head / a.group) * a.kh + r);
  }
  float v[VEC], o[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    v[j] = ok ? value(static_cast<const T*>(a.v), b * a.vb + (head / a.group) * a.vh + n0 + j) : 0.f;
    o[j] = 0.f;
  }
  float g2 = a.log_decay[head] * 1.44269504088896341f;
  g2 = g2 < -1e30f ? -1e30f : g2;
  const float lam = power(g2, 1);
  __syncthreads();
  for (int r0 = rl; r0 < a.K; r0 += RL * RB) {
    float s[RB][VEC];
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const int r = r0 + u * RL;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[u][j] = 0.f;
      if (ok && r < a.K && !cut) __builtin_memcpy(s[u], a.state + base + (int64_t)r * a.V, 4 * VEC);
    }
#pragma unroll
    for (int u = 0; u < RB; ++u) {
      const int r = r0 + u * RL;
      if (ok && r < a.K) {
        const float kr = sk[r], qr = sq[r];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s[u][j] = __fmaf_rn(kr, v[j], lam * s[u][j]);
          o[j] = __fmaf_rn(qr, s[u][j], o[j]);
        }
        __builtin_memcpy(a.state_out + base + (int64_t)r * a.V, s[u], 4 * VEC);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if constexpr (CL <= 32) o[j] = ppo::add_xor32(o[j]);
    if constexpr (CL <= 16) o[j] = ppo::add_xor16(o[j]);
    if constexpr (CL <= 8) o[j] += ppo::xor16<8>(o[j]);
    if ((tid & 63) < CL) part[tid >> 6][cl * VEC + j] = o[j];
  }
  __syncthreads();
  if (tid < CL * VEC && tid < a.slice) {
    const int n = slice * a.slice + tid;
    if (n < a.V) {
      const float s = ((part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid])) * a.scale;
      store4(static_cast<T*>(a.out) + bh * a.V + n, floatx4{s, s, s, s}, 1);
    }
  }
}

// ---- launches
constexpr int MAX_WIDTH = 128;

int padded(int K, int V) {
  const int w = std::max(K, V);
  return w <= 32 ? 32 : w <= 64 ? 64 : 128;
}

int chunk(int dtype) { return dtype == ATTN_F32 ? 32 : 64; }

// Pieces the step axis is cut into: enough workgroups to fill the chip, each
// of at least eight chunks (a piece's state is written and read back).
int segments_of(int dtype, int batch, int steps, int heads, int K, int V) {
  const int64_t pairs = std::max<int64_t>(1, (int64_t)batch * heads);
  const int c = chunk(dtype), D = padded(K, V);
  const int64_t want = 1024 * 64 / D / pairs, most = ppo::ceil_div(steps, 8 * c);
  const int segs = (int)std::max<int64_t>(1, std::min(want, most));
  const int seg_steps = ppo::ceil_div(ppo::ceil_div(std::max(steps, 1), segs), c) * c;
  return std::max(1, ppo::ceil_div(steps, seg_steps));
}

template <typename T, bool STATE>
void launch_width(hipStream_t st, const AttnArgs& a, int D, unsigned grid) {
  if (D == 32) hipLaunchKernelGGL((attention_kernel<T, 32, STATE>), dim3(grid), dim3(64), 0, st, a);
  else if (D == 64) hipLaunchKernelGGL((attention_kernel<T, 64, STATE>), dim3(grid), dim3(128), 0, st, a);
  else hipLaunchKernelGGL((attention_kernel<T, 128, STATE>), dim3(grid), dim3(256), 0, st, a);
}

// The pass from one direction's segments: their states from zeros, joined,
// then the outputs of every role.
void states_pass(hipStream_t st, int dtype, AttnArgs a, const Contraction& c, int batch) {
  if (a.segments == 1) return;
  a.role[0] = c;
  a.roles = 1;
  const int D = padded(c.x.width, c.z.width);
  const unsigned grid = (unsigned)((int64_t)batch * a.heads * (a.segments - 1));
  if (dtype == ATTN_F32) launch_width<float, true>(st, a, D, grid);
  else launch_width<uint16_t, true>(st, a, D, grid);
  const int64_t KV = (int64_t)c.x.width * c.z.width;
  hipLaunchKernelGGL(join_segments_kernel, dim3((unsigned)ppo::ceil_div64(KV, 256), (unsigned)(batch * a.heads)),
                     dim3(256), 0, st, c.states, a.factors, c.carry, KV, a.segments - 1);
}

void outputs_pass(hipStream_t st, int dtype, const AttnArgs& a, int batch) {
  const int D = padded(a.role[0].x.width, a.role[0].z.width);
  const unsigned grid = (unsigned)((int64_t)batch * a.heads * a.segments * a.roles);
  if (dtype == ATTN_F32) launch_width<float, false>(st, a, D, grid);
  else launch_width<uint16_t, false>(st, a, D, grid);
}

int check_sizes(const char* what, int dtype, int batch, int steps, int heads, int kv_heads, int K, int V) {
  if (dtype != ATTN_F32 && dtype != ATTN_BF16) return ppo::set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || heads < 0 || kv_heads < 0 || K < 0 || V < 0)
    return ppo::set_error(PPO_ERR_ARG, "%s: negative size (batch %d steps %d heads %d kv_heads %d widths %d %d)", what,
                          batch, steps, heads, kv_heads, K, V);
  if (K > MAX_WIDTH || V > MAX_WIDTH)
    return ppo::set_error(PPO_ERR_ARG, "%s: widths %d, %d above %d", what, K, V, MAX_WIDTH);
  if (heads > 0 && (kv_heads == 0 || heads % kv_heads))
    return ppo::set_error(PPO_ERR_ARG, "%s: %d heads do not share %d key heads evenly", what, heads, kv_heads);
  // the grid: four workgroups a head at most (four slices of a step, three outputs of the backward pass)
  if ((int64_t)batch * heads > (1 << 29) - 1)
    return ppo::set_error(PPO_ERR_ARG, "%s: batch x heads above %d", what, (1 << 29) - 1);
  return PPO_OK;
}

bool empty(int batch, int heads, int K, int V) { return batch == 0 || heads == 0 || K == 0 || V == 0; }

// A lane's byte within a chunk is counted in 32 bits.
int check_strides(const char* what, const int64_t* strides, int operands) {
  for (int i = 0; i < operands; ++i) {
    const int64_t st = strides[3 * i + 1];
    if (st < 0 || st > 1 << 23)
      return ppo::set_error(PPO_ERR_ARG, "%s: step stride %lld outside 0 .. %d", what, (long long)st, 1 << 23);
  }
  return PPO_OK;
}

int64_t state_floats(int dtype, int batch, int steps, int heads, int K, int V) {
  const int64_t more = segments_of(dtype, batch, steps, heads, K, V) - 1;
  return (int64_t)batch * heads * more * ((int64_t)K * V + 1);
}

AttnArgs common_args(int dtype, const float* log_decay, const uint8_t* done, const int32_t* lengths, int batch,
                     int steps, int heads, int K, int V) {
  AttnArgs a{};
  a.log_decay = log_decay;
  a.done = done;
  a.lengths = lengths;
  a.steps = steps;
  a.heads = heads;
  a.segments = segments_of(dtype, batch, steps, heads, K, V);
  const int c = chunk(dtype);
  a.seg_steps = ppo::ceil_div(ppo::ceil_div(std::max(steps, 1), a.segments), c) * c;
  return a;
}

}  // namespace

PPO_EXPORT int ppo_linear_attention_max_width(void) { return MAX_WIDTH; }

PPO_EXPORT size_t ppo_linear_attention_workspace(int dtype, int batch, int steps, int heads, int key_width,
                                                 int value_width) {
  if (check_sizes("ppo_linear_attention_workspace", dtype, batch, steps, heads, heads, key_width, value_width)) return 0;
  if (empty(batch, heads, key_width, value_width)) return 0;
  return sizeof(float) * (size_t)state_floats(dtype, batch, steps, heads, key_width, value_width);
}

PPO_EXPORT size_t ppo_linear_attention_bwd_workspace(int dtype, int batch, int steps, int heads, int kv_heads,
                                                     int key_width, int value_width) {
  if (check_sizes("ppo_linear_attention_bwd_workspace", dtype, batch, steps, heads, kv_heads, key_width, value_width))
    return 0;
  if (empty(batch, heads, key_width, value_width)) return 0;
  int64_t n = state_floats(dtype, batch, steps, heads, key_width, value_width);
  if (kv_heads < heads) n += (int64_t)batch * steps * heads * (key_width + value_width);
  return sizeof(float) * (size_t)n;
}

PPO_EXPORT int ppo_linear_attention_fwd(void* stream, int dtype, const void* q, const void* k, const void* v,
                                        const int64_t* strides, const float* log_decay, const float* carry,
                                        const uint8_t* done, const int32_t* lengths, float scale, void* out,
                                        float* final, void* workspace, size_t workspace_bytes, int batch, int steps,
                                        int heads, int kv_heads, int key_width, int value_width) {
  const char* what = "ppo_linear_attention_fwd";
  const int K = key_width, V = value_width;
  if (int rc = check_sizes(what, dtype, batch, steps, heads, kv_heads, K, V)) return rc;
  if (empty(batch, heads, K, V)) return PPO_OK;
  if (!log_decay || !final || !strides || (steps > 0 && (!q || !k || !v || !out)))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 3)) return rc;
  const int64_t floats = state_floats(dtype, batch, steps, heads, K, V);
  if (floats > 0 && (!workspace || workspace_bytes < sizeof(float) * (size_t)floats))
    return ppo::set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes,
                          sizeof(float) * (size_t)floats);
  AttnArgs a = common_args(dtype, log_decay, done, lengths, batch, steps, heads, K, V);
  float* states = static_cast<float*>(workspace);
  a.factors = states + (int64_t)batch * heads * (a.segments - 1) * K * V;
  const int group = heads / kv_heads;
  Contraction& c = a.role[0];
  c.x = Operand{q, strides[0], strides[1], strides[2], 1, K};
  c.y = Operand{k, strides[3], strides[4], strides[5], group, K};
  c.z = Operand{v, strides[6], strides[7], strides[8], group, V};
  c.out = out;
  c.carry = carry;
  c.states = states;
  c.final = final;
  c.intra = c.inter = scale;
  c.update = 1.f;
  a.roles = 1;
  states_pass(ppo::as_stream(stream), dtype, a, c, batch);
  outputs_pass(ppo::as_stream(stream), dtype, a, batch);
  return ppo::check_launch(what);
}

PPO_EXPORT int ppo_linear_attention_bwd(void* stream, int dtype, const void* q, const void* k, const void* v,
                                        const void* dout, const int64_t* strides, const float* log_decay,
                                        const float* carry, const uint8_t* done, const int32_t* lengths, float scale,
                                        const float* dfinal, const void* fwd_workspace, void* dq, void* dk, void* dv,
                                        float* dcarry, void* workspace, size_t workspace_bytes, int batch, int steps,
                                        int heads, int kv_heads, int key_width, int value_width) {
  const char* what = "ppo_linear_attention_bwd";
  const int K = key_width, V = value_width;
  if (int rc = check_sizes(what, dtype, batch, steps, heads, kv_heads, K, V)) return rc;
  if (empty(batch, heads, K, V)) return PPO_OK;
  if (!log_decay || !strides || (steps > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv)))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 4)) return rc;
  const int64_t floats = state_floats(dtype, batch, steps, heads, K, V);
  const size_t need = ppo_linear_attention_bwd_workspace(dtype, batch, steps, heads, kv_heads, K, V);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return ppo::set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  if (floats > 0 && !fwd_workspace) return ppo::set_error(PPO_ERR_ARG, "%s: null forward workspace", what);
  const int group = heads / kv_heads;
  AttnArgs a = common_args(dtype, log_decay, done, lengths, batch, steps, heads, K, V);
  float* states = static_cast<float*>(workspace);
  a.factors = states + (int64_t)batch * heads * (a.segments - 1) * K * V;
  float* wide = states + floats;
  float* wide_k = group > 1 ? wide : nullptr;
  float* wide_v = group > 1 ? wide + (int64_t)batch * steps * heads * K : nullptr;
  const Operand oq{q, strides[0], strides[1], strides[2], 1, K};
  const Operand ok{k, strides[3], strides[4], strides[5], group, K};
  const Operand ov{v, strides[6], strides[7], strides[8], group, V};
  const Operand od{dout, strides[9], strides[10], strides[11], 1, V};
  Contraction c{};
  // dv: the direction's states are D as they are
  c.x = ok;
  c.y = oq;
  c.z = od;
  c.out = group > 1 ? static_cast<void*>(wide_v) : dv;
  c.wide = group > 1;
  c.carry = dfinal;
  c.states = states;
  c.final = dcarry;
  c.backward = 1;
  c.intra = scale;
  c.inter = 1.f;
  c.update = scale;
  a.role[0] = c;
  // dk: the same states transposed
  c.x = ov;
  c.y = od;
  c.z = oq;
  c.out = group > 1 ? static_cast<void*>(wide_k) : dk;
  c.final = nullptr;
  c.transposed = 1;
  a.role[1] = c;
  // dq: the forward pass's states transposed
  c.x = od;
  c.y = ov;
  c.z = ok;
  c.out = dq;
  c.wide = 0;
  c.carry = carry;
  c.states = static_cast<float*>(const_cast<void*>(fwd_workspace));  // (read only)
  c.backward = 0;
  c.intra = c.inter = scale;
  c.update = 1.f;
  a.role[2] = c;
  a.roles = 3;
  states_pass(ppo::as_stream(stream), dtype, a, a.role[0], batch);
  outputs_pass(ppo::as_stream(stream), dtype, a, batch);
  if (group > 1 && steps > 0) {
    const int64_t rows = (int64_t)batch * steps * kv_heads;
    for (int i = 0; i < 2; ++i) {
      const int width = i ? V : K;
      const int64_t n = rows * width;
      const float* src = i ? wide_v : wide_k;
      void* dst = i ? dv : dk;
      const dim3 grid((unsigned)ppo::ceil_div64(n, 256));
      if (dtype == ATTN_F32)
        hipLaunchKernelGGL((sum_heads_kernel<float>), grid, dim3(256), 0, ppo::as_stream(stream), src,
                           static_cast<float*>(dst), n, width, group);
      else
        hipLaunchKernelGGL((sum_heads_kernel<uint16_t>), grid, dim3(256), 0, ppo::as_stream(stream), src,
                           static_cast<uint16_t*>(dst), n, width, group);
    }
  }
  return ppo::check_launch(what);
}

PPO_EXPORT int ppo_linear_attention_step(void* stream, int dtype, const void* q, const void* k, const void* v,
                                         const int64_t* strides, const float* log_decay, const uint8_t* done,
                                         const float* carry, float* final, void* out, float scale, int batch,
                                         int heads, int kv_heads, int key_width, int value_width) {
  const char* what = "ppo_linear_attention_step";
  const int K = key_width, V = value_width;
  if (int rc = check_sizes(what, dtype, batch, 1, heads, kv_heads, K, V)) return rc;
  if (empty(batch, heads, K, V)) return PPO_OK;
  if (!q || !k || !v || !strides || !log_decay || !carry || !final || !out)
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  StepArgs a{q, k, v, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], log_decay, done, carry,
             final, out, scale, heads, heads / kv_heads, K, V, 0, 0};
  // a workgroup a head, or slices of at least 32 columns where those are too
  // few to fill the chip
  const int64_t pairs = (int64_t)batch * heads;
  const bool vec = V % 4 == 0;
  int width = V > 64 && vec ? 128 : V > 32 ? 64 : 32;
  while (width > 32 && pairs * ppo::ceil_div(V, width) < 512) width /= 2;
  a.slice = width;
  a.slices = ppo::ceil_div(V, width);
  const dim3 grid((unsigned)(pairs * a.slices));
  hipStream_t st = ppo::as_stream(stream);
  auto launch = [&](auto t) {
    typedef decltype(t) T;
    if (vec) {
      if (width == 128) hipLaunchKernelGGL((attention_step_kernel<T, 4, 32>), grid, dim3(256), 0, st, a);
      else if (width == 64) hipLaunchKernelGGL((attention_step_kernel<T, 4, 16>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((attention_step_kernel<T, 4, 8>), grid, dim3(256), 0, st, a);
    } else {
      if (width == 64) hipLaunchKernelGGL((attention_step_kernel<T, 1, 64>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((attention_step_kernel<T, 1, 32>), grid, dim3(256), 0, st, a);
    }
  };
  if (dtype == ATTN_F32) launch(float());
  else launch(uint16_t());
  return ppo::check_launch(what);
}
