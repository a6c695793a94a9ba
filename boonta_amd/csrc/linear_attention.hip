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
  int streamed;             // the outputs are stored in whole rows past the caches
};

// ---- per type: chunks of 128 bytes of steps; a lane's MFMA operand of 16
// bytes (FR values).  One contraction block is 4 FR deep, a 16x16x32 bf16 MFMA
// or four 16x16x4 fp32 MFMAs: lane group g holds FR neighbouring values of it.
// An accumulator tile holds rows 4 g .. 4 g + 3 in group g, so a state tile is
// an operand over its rows without a move if slot 4 g + e of tile rt is row
//   bf16: 32 (rt / 2) + 8 g + 4 (rt % 2) + e    fp32: 16 rt + 4 g + e.
template <typename T> struct Type;

template <> struct Type<uint16_t> {
  typedef bf16x8 Frag;
  static constexpr int FR = 8, C = 64, PIECES = 3, PARTS = 2;
  static __device__ __forceinline__ constexpr int row(int rt, int slot) {
    return 32 * (rt >> 1) + 4 * (rt & 1) + 8 * (slot >> 2) + (slot & 3);
  }
  static __device__ __forceinline__ floatx4 mma(Frag a, Frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Type<float> {
  typedef floatx4 Frag;
  static constexpr int FR = 4, C = 32, PIECES = 1, PARTS = 1;
  static __device__ __forceinline__ constexpr int row(int rt, int slot) { return 16 * rt + slot; }
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

// The state as operands over its rows: contraction block kb, whose products
// are summed.  bf16: the state itself stays float32, and two pieces of it enter
// the product, as of the pair products: what they leave is at most 2^-17 of a
// term, where one bf16 would leave as much as the output's own rounding (outputs
// 2.4e-3 off in the norm in place of 1.7e-3).  (A second piece, against one:
// both passes of 128 x 1000 steps, 8 heads of 64, 432 -> 469 us, of 8 x 4096
// steps, 16 heads of 128, 611 -> 672; a third would gain nothing that an output
// in bf16 shows.)
template <int RT> __device__ __forceinline__ void state_frags(const floatx4 (&s)[RT], int kb, bf16x8 (&p)[2]) {
  floatx4 lo = s[2 * kb], hi = s[2 * kb + 1];
  p[0] = ppo::split_piece(lo, hi);
  p[1] = join(lo, hi);
}
template <int RT> __device__ __forceinline__ void state_frags(const floatx4 (&s)[RT], int kb, floatx4 (&p)[1]) {
  p[0] = s[kb];
}

// z times its steps' weights, as operands whose sum is the product to float32:
// one float32, or three bf16 pieces, each what the ones before leave (the
// states are float32 sums of exact products of these).
__device__ __forceinline__ void weigh(bf16x8 z, const float (&w)[8], bf16x8 (&p)[3], bool exact) {
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
  for (int i = 0; i < 2; ++i) p[i] = ppo::split_piece(lo, hi);
  if (exact) p[2] = join(lo, hi);
}
__device__ __forceinline__ void weigh(floatx4 z, const float (&w)[4], floatx4 (&p)[1], bool) {
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
// The same of the rows in slots l16 of state tile rt.
__device__ __forceinline__ int state_byte(int lane_byte, int rt, int tb, uint16_t) {
  return (lane_byte ^ (((4 * tb) ^ (2 * (rt & 1)) ^ (2 * (rt & 2))) << 4)) + (32 * (rt >> 1) + 4 * (rt & 1)) * 128;
}
__device__ __forceinline__ int state_byte(int lane_byte, int rt, int tb, float) { return tile_byte(lane_byte, rt, tb); }

// The same in a tile of rows of RB bytes, which repeat their banks every 1, 2
// or 4 rows: the XOR of row r's chunks, and the byte of an operand (row 16
// tile + l16, chunk 4 kb + g4).
template <int RB> __device__ __forceinline__ int row_swizzle(int r) {
  return RB % 256 == 0 ? r & 15 : RB % 128 == 0 ? swizzle(r) : (r >> 2) & 3;
}
template <int RB> __device__ __forceinline__ int row_byte(int l16, int g4, int tile, int kb) {
  const int lane_byte = l16 * RB + ((g4 ^ row_swizzle<RB>(l16)) << 4);
  const int at = tile * 16 * RB;
  if (RB % 256 == 0) return (lane_byte ^ ((kb & 3) << 6)) + (kb >> 2) * 256 + at;
  if (RB % 128 == 0) return (lane_byte ^ (((4 * (kb & 1)) ^ (2 * (tile & 3))) << 4)) + (kb >> 1) * 128 + at;
  return lane_byte + kb * 64 + at;
}

// Byte of chunk c of row ROWS group + e there, e < ROWS: the group's own with
// what e adds to the swizzle.
template <int RB, int ROWS> __device__ __forceinline__ int rows_byte(int c, int group, int e) {
  const int first = ROWS * group * RB + ((c ^ row_swizzle<RB>(ROWS * group)) << 4);
  return (first ^ (row_swizzle<RB>(e) << 4)) + e * RB;
}

// 16 bytes at a lane's 32-bit offset from an address that is uniform in the
// wave.  (Opaque, so that the sum stays in the load and each row of a lane
// costs one register, not an address.)
typedef __attribute__((address_space(1))) const char* GlobalBytes;

__device__ __forceinline__ GlobalBytes uniform(const void* p) {
  uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p);
  uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)p >> 32));
  asm("" : "+s"(lo), "+s"(hi));
  return (GlobalBytes)((uintptr_t)hi << 32 | lo);
}
__device__ __forceinline__ uint4 load_chunk(GlobalBytes base, uint32_t byte) {
  typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
  const word4 v = *(__attribute__((address_space(1))) const word4*)(base + byte);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A chunk of 16 bytes (elements c0 ..) with what is past the row's `width`
// zeros: the last chunk of a width that FR does not divide was read from its
// end, so that no load leaves the row, and is shifted.
template <typename T>
__device__ __forceinline__ uint4 trim_chunk(uint4 v, int c0, int width) {
  constexpr int FR = Type<T>::FR;
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

// Four steps' chunks (columns FR dc .. of steps 4 tg ..) as columns: element j
// of the chunk over the four steps, at a byte of the lane's with j's row and
// what j adds to the swizzle.
__device__ __forceinline__ int transposed_byte(int dc, int tg, uint16_t) {
  return dc * 1024 + ((((tg >> 1) ^ (4 * (dc & 1)) ^ dc) & 7) << 4) + ((tg & 1) << 3);
}
__device__ __forceinline__ int transposed_byte(int dc, int tg, float) {
  return dc * 512 + (((tg ^ (2 * dc) ^ (dc >> 1)) & 7) << 4);
}
__device__ __forceinline__ void write_transposed(char* t, int byte, const uint4 (&v)[4], uint16_t) {
  const uint32_t q[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w},
                            {v[1].x, v[1].y, v[1].z, v[1].w},
                            {v[2].x, v[2].y, v[2].z, v[2].w},
                            {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;  // the high or low half of two words
    *reinterpret_cast<uint2*>(t + (byte ^ ((j >> 1) << 4)) + j * 128) =
        make_uint2(__builtin_amdgcn_perm(q[1][j >> 1], q[0][j >> 1], sel),
                   __builtin_amdgcn_perm(q[3][j >> 1], q[2][j >> 1], sel));
  }
}
__device__ __forceinline__ void write_transposed(char* t, int byte, const uint4 (&v)[4], float) {
  *reinterpret_cast<uint4*>(t + byte) = make_uint4(v[0].x, v[1].x, v[2].x, v[3].x);
  *reinterpret_cast<uint4*>(t + byte + 128) = make_uint4(v[0].y, v[1].y, v[2].y, v[3].y);
  *reinterpret_cast<uint4*>(t + (byte ^ 16) + 256) = make_uint4(v[0].z, v[1].z, v[2].z, v[3].z);
  *reinterpret_cast<uint4*>(t + (byte ^ 16) + 384) = make_uint4(v[0].w, v[1].w, v[2].w, v[3].w);
}

typedef __attribute__((address_space(1))) char* GlobalOut;
typedef float floatx4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Four consecutive outputs of a row, `left` of them inside it.
__device__ __forceinline__ void store4(GlobalOut p, floatx4 v, int left, uint16_t) {
  typedef __attribute__((address_space(1))) uint16_t* Out;
  typedef uint32_t word2 __attribute__((ext_vector_type(2), aligned(2)));
  const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
  if (left >= 4) {
    *(__attribute__((address_space(1))) word2*)p = word2{lo, hi};
  } else {
    if (left > 0) ((Out)p)[0] = (uint16_t)lo;
    if (left > 1) ((Out)p)[1] = (uint16_t)(lo >> 16);
    if (left > 2) ((Out)p)[2] = (uint16_t)hi;
  }
}
__device__ __forceinline__ void store4(GlobalOut p, floatx4 v, int left, float) {
  typedef __attribute__((address_space(1))) float* Out;
  if (left >= 4) {
    *(__attribute__((address_space(1))) floatx4_a4*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) ((Out)p)[e] = v[e];
  }
}
// A chunk of 16 bytes of a row of T, `left` elements inside it, past the caches.
template <typename T> __device__ __forceinline__ void stream_chunk(GlobalOut p, uint4 v, int left) {
  typedef __attribute__((address_space(1))) uint16_t* Halves;
  typedef __attribute__((address_space(1))) uint32_t* Words;
  typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
  const word4 w = {v.x, v.y, v.z, v.w};
  if (left >= Type<T>::FR) {
    __builtin_nontemporal_store(w, (__attribute__((address_space(1))) word4*)p);
  } else {
#pragma unroll
    for (int e = 0; e < Type<T>::FR - 1; ++e)
      if (e < left) {
        if constexpr (sizeof(T) == 2) ((Halves)p)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
        else ((Words)p)[e] = w[e];
      }
  }
}
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = (uint16_t)pack_bf16(v, v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// The value, as if computed here: what depends on it is not moved out of the
// loop, where it would hold registers for a part that is seldom run.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Waits for this wave's loads: before the streamed stores, and where a chunk
// begins without them, since what is waited for later counts the stores too.
// (Without, products of one piece: both passes of 128 x 1000 steps, 8 heads of
// 64, 431 -> 435 us, float32 ones of 4 x 4000 steps, 4 heads of 128, 317 -> 321.)
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // (no other counter)

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// x, or zero (a select: as a branch, each load before it would wait alone)
__device__ __forceinline__ float keep_if(float x, bool keep) { return keep ? x : 0.f; }

// A value every lane of the wave has, in a scalar register.
__device__ __forceinline__ float same(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

__device__ __forceinline__ float power(float g2, int e) { return __builtin_amdgcn_exp2f(g2 * (float)e); }

// One workgroup per (role, head, segment, sequence): D / 16 waves, each with
// 16 columns of the D x D state in its accumulators.  Widths below D are
// padded with zeros.  Each chunk of x, y, z is loaded once, a chunk ahead, into
// registers, and laid out in LDS by rows (x, y: the pair products) and by
// columns (y, z: contractions over steps).  STATE: only the state, from zeros,
// for the segments before the last.
// Sixteen columns a wave keep a 128 x 128 state, the chunk ahead and the
// products' operands in 128 registers, four waves a SIMD: 64-wide bf16 takes
// 40 KB of LDS, four workgroups a CU, 128-wide 79 KB, two.  Bound by HBM and a
// chunk's vector and LDS work together.  Measured (traces of calls one after
// the other, operands of three sets in turn), bf16: 128 x 1000 steps, 8 heads of
// 64 with resets, forward 136 us (558 MB, 4.1 TB/s), backward 340 (1.32 GB, 3.9
// TB/s); 65536 steps, 16 heads of 128, states 121 us (553 MB, 4.6 TB/s) and
// outputs 287 (1.12 GB, 3.9 TB/s); 8 x 4096 steps, 16 heads of 128, states 57 us
// (227 MB: one and a half workgroups a CU, bound by instructions), outputs 144,
// backward 392 (1.46 GB, 3.7 TB/s, vector instructions issuing 60 % of the time,
// matrix units busy 31 %).  float32, 256 x 64 steps, 4 heads of 64: 30 us, a
// third of it matrix products (16x16x4), backward 68.
template <typename T, int D, bool STATE>
__global__ void __launch_bounds__(4 * D, D == 96 ? 2 : D == 32 ? 3 : 4) attention_kernel(AttnArgs p) {
  typedef typename Type<T>::Frag Frag;
  constexpr int FR = Type<T>::FR, C = Type<T>::C, W = D / 16, KB = D / (4 * FR), RT = D / 16, QT = C / 16;
  constexpr int PIECES = Type<T>::PIECES, PARTS = Type<T>::PARTS, TILES = QT * (QT + 1) / 2;
  constexpr int RB = D * (int)sizeof(T), ROWS = C * RB, COLS = D * 128, PAIRS = C * 96;
  // The pair products' second pieces: after the first ones, or, where that would
  // leave a workgroup less a CU (64-wide: 46 KB; 128 x 1000 steps, 8 heads,
  // forward 137 -> 156 us, backward 333 -> 350), in place of y's rows (and what
  // those lack) once the pair products are formed.
  constexpr bool OVER_Y = PARTS == 2 && D <= 64;
  constexpr int MORE = !OVER_Y ? (PARTS - 1) * PAIRS : ROWS < PAIRS ? PAIRS - ROWS : 0;
  // Streamed outputs go through LDS to be stored in whole rows.  (96-wide, rows
  // of one and a half lines and few waves, products of one piece: 175 -> 181 us, so
  // not there.)
  constexpr bool ROWS_OUT = !STATE && D != 96;
  // y and z by columns, x and y by rows, and the pair products: all queries
  // with the chunk's first half of keys, the later half with the other
  __shared__ __attribute__((aligned(16))) char smem[(STATE ? 0 : 2 * ROWS + MORE + PAIRS) + 2 * COLS];
  __shared__ __attribute__((aligned(16))) float weights[C];  // of the chunk's steps in the state after it
  __shared__ float reaches[C];                               // factors of x St
  __shared__ float powers[16 + C];                           // intra lam^d at 16 + d
  __shared__ int odd[2];
  char* const yt = smem;
  char* const zt = smem + COLS;
  char* const xr = smem + 2 * COLS;
  char* const yr = smem + 2 * COLS + ROWS;
  char* const pr = smem + 2 * COLS + 2 * ROWS + (OVER_Y ? MORE : 0);
  char* const pr_low = OVER_Y ? yr : pr + PAIRS;

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  const bool streamed = ROWS_OUT && p.streamed && !c.wide;
  const bool back = c.backward;
  const int col = 16 * wave + l16;  // this lane's column of the state

  const int len = p.lengths ? min(max(p.lengths[b], 0), p.steps) : p.steps;
  float g2 = p.log_decay[head] * 1.44269504088896341f;
  g2 = same(g2 < -1e30f ? -1e30f : g2);  // (a decay of zero: 0 times an infinite exponent is no number)
  const uint8_t* done = p.done ? p.done + (int64_t)b * p.steps : nullptr;
  const int first = seg * p.seg_steps;                                        // steps in the order of processing
  const int last = min(len, first + p.seg_steps);
  const int pitch_o = p.heads * N;  // (at most 2^23)
  const int64_t base_o = ((int64_t)b * p.steps * p.heads + head) * N;

  // rows past the sequence's end hold zeros
  if constexpr (!STATE) {
    const int end = min(p.steps, first + p.seg_steps);
    for (int t = max(len, first) + wave; t < end; t += W)
      for (int n = lane; n < N; n += 64) {
        if (c.wide) static_cast<float*>(c.out)[base_o + (int64_t)t * pitch_o + n] = 0.f;
        else static_cast<T*>(c.out)[base_o + (int64_t)t * pitch_o + n] = T(0);
      }
  }

  // a thread's share of a chunk: of y (the first half of the waves) or z four
  // steps' chunks of columns, of x two steps'
  const bool second = wave >= W / 2;
  const Operand& oyz = second ? c.z : c.y;
  const T* xp = static_cast<const T*>(c.x.p) + b * c.x.sb + (head / c.x.group) * c.x.sh;
  const T* yzp = static_cast<const T*>(oyz.p) + b * oyz.sb + (head / oyz.group) * oyz.sh;
  uint4 rx[2], ryz[4];
  auto fetch = [&](auto& v, const Operand& o, const T* base, int r0, int chunk, int step) {
    constexpr int ROWS_ = sizeof(v) / 16;
    const int st = (int)o.st, at = min(chunk * FR, o.width - FR), count = min(C, last - r0);
    const GlobalBytes low = uniform(base + (int64_t)(back ? len - r0 - count : r0) * st);
    uint32_t byte[ROWS_];
    if (count == C) {
      const uint32_t next = (uint32_t)((back ? -st : st) * (int)sizeof(T));
      byte[0] = (uint32_t)((back ? C - 1 - step : step) * st + at) * (uint32_t)sizeof(T);
#pragma unroll
      for (int e = 1; e < ROWS_; ++e) byte[e] = byte[e - 1] + next;
    } else {
#pragma unroll
      for (int e = 0; e < ROWS_; ++e) {
        const int s = min(step + e, count - 1);
        byte[e] = (uint32_t)((back ? count - 1 - s : s) * st + at) * (uint32_t)sizeof(T);
      }
    }
#pragma unroll
    for (int e = 0; e < ROWS_; ++e) v[e] = load_chunk(low, byte[e]);
  };
  auto finish = [&](auto& v, int width, int n, int chunk, int step) {
    constexpr int ROWS_ = sizeof(v) / 16;
    if (width < D) {
      const int c0 = here(chunk * FR);
#pragma unroll
      for (int e = 0; e < ROWS_; ++e) v[e] = trim_chunk<T>(v[e], c0, width);
    }
    if (n < C) {
      const int s = here(step);
#pragma unroll
      for (int e = 0; e < ROWS_; ++e)
        if (s + e >= n) v[e] = make_uint4(0, 0, 0, 0);
    }
  };
  auto fetch_done = [&](int r0, int lane) -> int {  // whether the state entering step r0 + lane is dropped
    const int s = r0 + lane;
    if (!done || lane >= C || s >= last) return 0;
    if (!back) return done[s];
    return s > 0 ? done[len - s] : 0;
  };
  int cut_next = 0;
  auto fetch_all = [&](int r0, int tid) {
    const uint32_t unit = second ? tid - 2 * D : tid, chunks = D / FR;
    if constexpr (!STATE) fetch(rx, c.x, xp, r0, (uint32_t)tid % chunks, 2 * ((uint32_t)tid / chunks));
    fetch(ryz, oyz, yzp, r0, unit % chunks, 4 * (unit / chunks));
    cut_next = fetch_done(r0, tid & 63);
  };
  // (STATE goes from the segment's last chunk to its first)
  int r0 = STATE && first < last ? first + (last - first - 1) / C * C : first, it = 0;
  if (first < last) fetch_all(r0, tid);

  // the state entering the segment: rows 16 rt + 4 g4 + e of column col
  floatx4 S[RT];
  const float* entry = nullptr;
  if constexpr (!STATE) entry = seg == 0 ? (c.carry ? c.carry + bh * KV : nullptr)
                                         : c.states + (bh * (p.segments - 1) + seg - 1) * KV;
  const int pitch_r = c.transposed ? 1 : N, pitch_n = c.transposed ? R : 1;  // of the state in memory
  if (entry) {
    const int at_n = min(col, N - 1) * pitch_n;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[rt][e] = entry[at_n + min(Type<T>::row(rt, 4 * g4 + e), R - 1) * pitch_r];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[rt][e] = Type<T>::row(rt, 4 * g4 + e) < R && col < N ? S[rt][e] : 0.f;
  } else {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) S[rt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  if (tid < 2) odd[tid] = 0;
  if (tid < 16 + C) powers[tid] = tid < 16 ? 0.f : c.intra * power(g2, tid - 16);
  if constexpr (!STATE)
    for (int i = tid; i < (MORE + PAIRS) / 16; i += 4 * D)
      reinterpret_cast<uint4*>(smem + 2 * COLS + 2 * ROWS)[i] = make_uint4(0, 0, 0, 0);
  lds_barrier();

  // Whether the state itself is an output (or, STATE, leads to one): the third
  // piece of its terms (2^-17 of them) is no more than what a state loses that
  // only enters products, in two pieces.  With it, 16 heads of 128: 65536 steps
  // 407 -> 421 us, both passes of 8 x 4096 steps 672 -> 702 us.
  const bool exact = c.final && (STATE || seg == p.segments - 1);
  uint64_t cut = 0;   // the chunk's steps that drop the state
  // Lays out steps r0 .. r0 + n - 1, as loaded, and loads the chunk from `next` (>= 0) on.
  // Whether y or z holds an infinity or NaN.  (Here and below a lane's places
  // are formed in every chunk: kept, they would spill.)
  auto stage = [&](int n, int next) -> bool {
    const int tid = here(threadIdx.x), lane = tid & 63;
    const uint32_t unit = second ? tid - 2 * D : tid, chunks = D / FR;
    const int dc = unit % chunks, tg = unit / chunks, dx = (uint32_t)tid % chunks, tx = (uint32_t)tid / chunks;
    // a backward sequence's first step takes the state as it is
    const int skip = back && r0 == 0 ? 1 : 0;
    cut = __ballot(cut_next != 0 && lane < n);
    if constexpr (!STATE) finish(rx, R, n, dx, 2 * tx);
    finish(ryz, second ? N : R, n, dc, 4 * tg);
    bool is_odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) is_odd |= odd_exponent(ryz[e], T());
    if (__ballot(is_odd) && lane == 0) odd[it & 1] = 1;
    if constexpr (!STATE) {
#pragma unroll
      for (int e = 0; e < 2; ++e) *reinterpret_cast<uint4*>(xr + rows_byte<RB, 2>(dx, tx, e)) = rx[e];
    }
    const int columns_byte = transposed_byte(dc, tg, T());
    if (second) {
      write_transposed(zt, columns_byte, ryz, T());
    } else {
      if constexpr (!STATE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(yr + rows_byte<RB, 4>(dc, tg, e)) = ryz[e];
      }
      write_transposed(yt, columns_byte, ryz, T());
    }
    if (wave == 0 && lane < C) {
      const int last_cut = cut ? 63 - __clzll(cut) : -1;
      const int left = (STATE ? last - r0 : n) - 1 - lane;
      weights[lane] = lane < n && lane >= last_cut ? c.update * power(g2, left) : 0.f;
      if (!STATE) reaches[lane] = (cut & (~0ull >> (63 - lane))) == 0 ? c.inter * power(g2, lane + 1 - skip) : 0.f;
    }
    if (next >= 0) fetch_all(next, tid);
    lds_barrier();
    const bool is_bad = __builtin_amdgcn_readfirstlane(odd[it & 1]);
    if (tid == 0) odd[(it + 1) & 1] = 0;
    ++it;
    return is_bad;
  };
  auto chunk = [&](int n) {
    // (the products before another workgroup's laying out: 16 heads of 128, both passes of 8 x 4096 steps 681 ->
    // 672 us, 65536 steps 422 -> 407 us)
    __builtin_amdgcn_s_setprio(1);
    const int tid = here(threadIdx.x), lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
    const int skip = back && r0 == 0 ? 1 : 0;
    const float fade = STATE ? 1.f : same(power(g2, n - skip));
    const int lane_byte = l16 * 128 + ((g4 ^ swizzle(l16)) << 4);
    {
      if constexpr (!STATE) {
        // pair products, keys as rows so that a lane holds four keys of one
        // query: tile (qt, kt) of the lower triangle, dealt to the waves
        const int pair_byte = l16 * 64 + ((g4 ^ (l16 >> 2)) << 4);
        // (0, 0), (1, 0), (1, 1), ..: two bits a tile
        auto query_tile = [](int idx) { return (int)(0xffa94u >> (2 * idx) & 3); };
        auto key_tile = [](int idx) { return (int)(0xe4910u >> (2 * idx) & 3); };
        auto half_byte = [&](int qt, int kt) {  // bf16: of this lane's four keys
          const int chunk = 2 * (kt & 1) + (g4 >> 1);
          return l16 * 64 + ((chunk ^ (l16 >> 2)) << 4) + ((g4 & 1) << 3) + qt * 1024 + (kt >> 1) * C * 32;
        };
        auto pair = [&](int idx, uint2& low) {  // low: the second pieces, where they are written later
          const int qt = query_tile(idx), kt = key_tile(idx);
          floatx4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const Frag ya = *reinterpret_cast<const Frag*>(yr + row_byte<RB>(l16, g4, kt, kb));
            const Frag xb = *reinterpret_cast<const Frag*>(xr + row_byte<RB>(l16, g4, qt, kb));
            a = Type<T>::mma(ya, xb, a);
          }
          const int i = 16 * qt + l16, j0 = 16 * kt + 4 * g4;
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] *= powers[16 + i - j0 - e];
          if (cut) {
            const uint64_t upto = cut & (~0ull >> (63 - i));
            const int from = upto ? 63 - __clzll(upto) : 0;  // the last reset up to step i
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = keep_if(a[e], j0 + e >= from);
          }
          if (kt == qt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = keep_if(a[e], j0 + e <= i);
          }
          if constexpr (PARTS == 2) {
            const int at = half_byte(qt, kt);
            const uint32_t u = pack_bf16(a[0], a[1]), w = pack_bf16(a[2], a[3]);
            *reinterpret_cast<uint2*>(pr + at) = make_uint2(u, w);
            a[0] -= __uint_as_float(u << 16);
            a[1] -= __uint_as_float(u & 0xffff0000u);
            a[2] -= __uint_as_float(w << 16);
            a[3] -= __uint_as_float(w & 0xffff0000u);
            low = make_uint2(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]));
            if constexpr (!OVER_Y) *reinterpret_cast<uint2*>(pr_low + at) = low;
          } else {
            *reinterpret_cast<floatx4*>(pr + pair_byte + qt * 1024 + kt * C * 32) = a;
          }
        };
        if constexpr (OVER_Y) {
          constexpr int DEALT = (TILES + W - 1) / W;
          uint2 low[DEALT];
#pragma unroll
          for (int i = 0; i < DEALT; ++i)
            if (wave + i * W < TILES) pair(wave + i * W, low[i]);
          lds_barrier();
#pragma unroll
          for (int i = 0; i < DEALT; ++i)
            if (wave + i * W < TILES) {
              const int qt = query_tile(wave + i * W), kt = key_tile(wave + i * W);
              *reinterpret_cast<uint2*>(pr_low + half_byte(qt, kt)) = low[i];
              // the masked tile that the products take with an even diagonal one (of the first pieces it stays zero)
              if (kt == qt && !(kt & 1)) *reinterpret_cast<uint2*>(pr_low + half_byte(qt, kt + 1)) = make_uint2(0, 0);
            }
        } else {
          uint2 low;
#pragma unroll 1
          for (int idx = wave; idx < TILES; idx += W) pair(idx, low);
        }
        // x times the entry state (rows: its columns)
        floatx4 acc[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) acc[qt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Frag s[PARTS], x[QT];
          state_frags(S, kb, s);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) x[qt] = *reinterpret_cast<const Frag*>(xr + row_byte<RB>(l16, g4, qt, kb));
#pragma unroll
          for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) acc[qt] = Type<T>::mma(s[q], x[qt], acc[qt]);
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const float f = reaches[16 * qt + l16];
          if (cut) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[qt][e] = (cut & (~0ull >> (63 - (16 * qt + l16)))) == 0 ? acc[qt][e] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[qt][e] *= f;
        }
        lds_barrier();
        // the pair products times z, and the outputs
        Frag z[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) z[tb] = *reinterpret_cast<const Frag*>(zt + tile_byte(lane_byte, wave, tb));
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q) {
          const char* const a = (q ? pr_low : pr) + pair_byte;
#pragma unroll
          for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              if (16 * qt + 15 < 4 * FR * tb) continue;  // keys after the queries
              acc[qt] = Type<T>::mma(z[tb], *reinterpret_cast<const Frag*>(a + qt * 1024 + tb * C * 32), acc[qt]);
            }
        }
        if (!streamed) {
          const int size = c.wide ? 4 : (int)sizeof(T), n0 = 16 * wave + 4 * g4;
          const GlobalOut low = (GlobalOut)uniform(static_cast<const char*>(c.out) +
                                                   (base_o + (back ? len - r0 - n : r0) * (int64_t)pitch_o) * size);
          uint32_t byte = (uint32_t)((back ? n - 1 - l16 : l16) * pitch_o + n0) * size;
          const uint32_t next = (uint32_t)((back ? -16 : 16) * pitch_o * size);
          if (n == C && 16 * wave + 16 <= N && !c.wide) {  // (without the tests: 96-wide 180 -> 175 us)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt, byte += next) store4(low + byte, acc[qt], 4, T());
          } else {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt, byte += next) {
              if (16 * qt + l16 < n) {
                if (c.wide) store4(low + byte, acc[qt], N - n0, float());
                else store4(low + byte, acc[qt], N - n0, T());
              }
            }
          }
        } else {
          // for whole rows: in place of x, which no wave reads any more
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            if constexpr (sizeof(T) == 2) {
              *reinterpret_cast<uint2*>(xr + row_byte<RB>(l16, 2 * (wave & 1) + (g4 >> 1), qt, wave >> 1) +
                                        ((g4 & 1) << 3)) =
                  make_uint2(pack_bf16(acc[qt][0], acc[qt][1]), pack_bf16(acc[qt][2], acc[qt][3]));
            } else {
              *reinterpret_cast<floatx4*>(xr + row_byte<RB>(l16, g4, qt, wave)) = acc[qt];
            }
          }
        }
      }
      // state: its rows by y's columns, contracted over the steps (from zeros
      // every step's weight is that at the segment's end)
      const int slot_row = Type<T>::row(0, l16), state_lane_byte = slot_row * 128 + ((g4 ^ swizzle(slot_row)) << 4);
      if constexpr (!STATE) {
        if (cut) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) S[rt] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[rt][e] *= fade;
      }
#pragma unroll
      for (int tb = 0; tb < 2; ++tb) {
        float weight[FR];
#pragma unroll
        for (int e = 0; e < FR; e += 4)
          *reinterpret_cast<floatx4*>(weight + e) =
              *reinterpret_cast<const floatx4*>(weights + 4 * FR * tb + FR * g4 + e);
        Frag w[PIECES];
        weigh(*reinterpret_cast<const Frag*>(zt + tile_byte(lane_byte, wave, tb)), weight, w, exact);
        // (in groups, so that products of one accumulator do not wait for each
        // other and no more operands are ahead than fit)
        constexpr int GROUP = RT % 4 == 0 ? 4 : RT % 3 == 0 ? 3 : 2;
#pragma unroll
        for (int r4 = 0; r4 < RT; r4 += GROUP) {
          if (D == 128) __builtin_amdgcn_sched_barrier(0);
          Frag ya[GROUP];
#pragma unroll
          for (int i = 0; i < GROUP; ++i)
            ya[i] = *reinterpret_cast<const Frag*>(yt + state_byte(state_lane_byte, r4 + i, tb, T()));
#pragma unroll
          for (int q = PIECES - 1; q >= 0; --q) {
            if (q == 2 && !exact) continue;
#pragma unroll
            for (int i = 0; i < GROUP; ++i) S[r4 + i] = Type<T>::mma(ya[i], w[q], S[r4 + i]);
          }
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    lds_barrier();
    if (!streamed) return;
    // whole rows of outputs, from where this thread lays out x next
    const int dx = (uint32_t)tid % (D / FR), tx = (uint32_t)tid / (D / FR), left = N - dx * FR;
    const GlobalOut low = (GlobalOut)uniform(static_cast<const T*>(c.out) + base_o +
                                             (back ? len - r0 - n : r0) * (int64_t)pitch_o);
    uint4 v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = *reinterpret_cast<const uint4*>(xr + rows_byte<RB, 2>(dx, tx, e));
    loads_done();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = 2 * tx + e, at = (back ? n - 1 - row : row) * pitch_o + dx * FR;
      if (row < n) stream_chunk<T>(low + (uint32_t)at * (uint32_t)sizeof(T), v[e], left);
    }
  };
  // The products multiply a masked pair by zero, which an infinity or NaN in y or
  // z outlasts: the steps of such a chunk are taken one by one.  (Padding stays
  // zero: a zero times an infinity is none.)
  auto clear_padding = [&]() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (Type<T>::row(rt, 4 * g4 + e) >= R) S[rt][e] = 0.f;
  };
  if constexpr (!STATE) {
    while (r0 < last) {
      bool is_bad = false;
      loads_done();
      while (r0 < last) {
        const int n = min(C, last - r0);
        is_bad = stage(n, r0 + n < last ? r0 + n : -1);
        if (__builtin_expect(is_bad, 0)) {
          loads_done();
          break;
        }
        chunk(n);
        r0 += n;
      }
      if (__builtin_expect(is_bad, 0)) {
        const int end = min(last, r0 + C);
#pragma unroll 1
        while (r0 < end) {
          lds_barrier();
          fetch_all(r0, tid);
          stage(1, r0 + 1 < last ? r0 + 1 : -1);
          chunk(1);
          r0 += 1;
          clear_padding();
        }
      }
    }
  } else {
    // From the segment's last chunk to its first, or to the last reset: what is
    // before it reaches no state after the segment.  (And what the outputs'
    // launch reads first is what this one read last.)
    bool reset = false;
    while (r0 >= first && first < last && !reset) {
      bool is_bad = false;
      while (r0 >= first && !reset) {
        const int n = min(C, last - r0);
        is_bad = stage(n, r0 > first ? r0 - C : -1);
        if (__builtin_expect(is_bad, 0)) break;
        chunk(n);
        reset = cut != 0;
        r0 -= C;
      }
      if (__builtin_expect(is_bad, 0)) {
        const int low = r0;
        r0 = min(low + C, last);
#pragma unroll 1
        while (r0 > low && !reset) {
          lds_barrier();
          r0 -= 1;
          fetch_all(r0, tid);
          stage(1, -1);
          chunk(1);
          reset = cut != 0;
          clear_padding();
        }
        r0 = low - C;
        lds_barrier();
        if (r0 >= first) fetch_all(r0, tid);
      }
    }
    if (tid == 0)
      p.factors[bh * (p.segments - 1) + seg] =
          reset ? -1.f : power(g2, max(last - first, 0) - (back && first == 0 && last > 0 ? 1 : 0));
  }

  float* exit = STATE ? c.states + (bh * (p.segments - 1) + seg) * KV
                      : (c.final && seg == p.segments - 1 ? c.final + bh * KV : nullptr);
  if (!exit) return;
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
    for (int e = 0; e < 4; ++e) {
      const int r = Type<T>::row(rt, 4 * g4 + e);
      if (r < R && col < N) exit[r * pitch_r + col * pitch_n] = drop ? 0.f : S[rt][e] * f;
    }
}

// The states entering each segment after the first, from what each segment
// before the last adds from zeros and how it fades what enters it; in place.
// Four neighbouring values a thread (a state's last ones apart), four segments'
// loads in flight; bound by HBM, or by its launch: 128 pairs of 3 states of
// 128 x 128 take 9 to 11 us (50 MB, 5 TB/s), 192 of 4 of 64 x 64 6 us.
__global__ void __launch_bounds__(64) join_segments_kernel(float* states, const float* factors, const float* carry,
                                                            int KV, int segs) {
  const int i = (blockIdx.x * 64 + threadIdx.x) * 4, left = KV - i;
  const int64_t bh = blockIdx.y;
  if (left <= 0) return;
  auto load = [&](const float* p) -> floatx4 {
    if (left >= 4) return *reinterpret_cast<const floatx4_a4*>(p);
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < left; ++e) v[e] = p[e];
    return v;
  };
  floatx4 s = carry ? load(carry + bh * KV + i) : floatx4{0.f, 0.f, 0.f, 0.f};
  float* p = states + bh * segs * KV + i;
  const float* f = factors + bh * segs;
  constexpr int U = 4;
  for (int k0 = 0; k0 < segs; k0 += U) {
    floatx4 v[U];
    float fade[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      v[k] = load(p + (int64_t)min(k0 + k, segs - 1) * KV);
      fade[k] = f[min(k0 + k, segs - 1)];
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (k0 + k < segs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = fade[k] < 0.f ? v[k][e] : __fmaf_rn(fade[k], s[e], v[k][e]);
        store4((GlobalOut)(p + (int64_t)(k0 + k) * KV), s, left, float());
      }
  }
}

// Gradients of heads that `group` query heads share: their sum.
template <typename T>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* x, T* out, int64_t n, int width, int group) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const float* p = x + i / width * width * group + i % width;
    float s = 0.f;
    for (int j = 0; j < group; ++j) s += p[(int64_t)j * width];
    store1(out + i, s);
  }
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
// is read and written once; bound by HBM: 1024 x 8 heads of 128 take 205 us,
// 5.3 TB/s (16 x 4 heads of 64 take 4.4 us, a launch's own time).
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
      store1(static_cast<T*>(a.out) + bh * a.V + n, s);
    }
  }
}

// ---- launches
constexpr int MAX_WIDTH = 128;

// The width of a launch.  96 of its own, batch 8, 4096 steps, 16 heads against
// padded to 128: bf16 188 us (199) forward and 627 (632) with the backward,
// batch 2, 512 steps, 4 heads of 80 23.7 us (27.0); float32, 2048 steps, 229 us
// (300).
int padded(int K, int V) {
  const int w = std::max(K, V);
  return w <= 32 ? 32 : w <= 64 ? 64 : w <= 96 ? 96 : 128;
}

int chunk(int dtype) { return dtype == ATTN_F32 ? 32 : 64; }

// Segments the step axis is cut into: as many workgroups as the chip's 256 CUs
// hold at a time (16 waves each), while a segment keeps two chunks or more,
// since its state is written, joined and read back.  Measured, bf16: against
// half and twice as many, batch 1, 65536 steps, 16 heads of 128 takes 407 us
// (468, 434) and both passes of batch 8, 4096 steps, 16 heads of 128 take 672
// us (712, 740); against segments of four chunks, batch 4, 2048 steps, 8 heads
// of 64 takes 31.4 us (34.1).
int segments_of(int dtype, int batch, int steps, int heads, int K, int V) {
  const int64_t pairs = std::max<int64_t>(1, (int64_t)batch * heads);
  const int c = chunk(dtype), D = padded(K, V);
  const int64_t want = 256 * (256 / D) / pairs, most = ppo::ceil_div(steps, 2 * c);
  const int segs = (int)std::max<int64_t>(1, std::min(want, most));
  const int seg_steps = ppo::ceil_div(ppo::ceil_div(std::max(steps, 1), segs), c) * c;
  return std::max(1, ppo::ceil_div(steps, seg_steps));
}

template <typename T, bool STATE>
void launch_width(hipStream_t st, const AttnArgs& a, int D, unsigned grid) {
  if (D == 32) hipLaunchKernelGGL((attention_kernel<T, 32, STATE>), dim3(grid), dim3(128), 0, st, a);
  else if (D == 64) hipLaunchKernelGGL((attention_kernel<T, 64, STATE>), dim3(grid), dim3(256), 0, st, a);
  else if (D == 96) hipLaunchKernelGGL((attention_kernel<T, 96, STATE>), dim3(grid), dim3(384), 0, st, a);
  else hipLaunchKernelGGL((attention_kernel<T, 128, STATE>), dim3(grid), dim3(512), 0, st, a);
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
  const int KV = c.x.width * c.z.width;
  hipLaunchKernelGGL(join_segments_kernel, dim3((unsigned)ppo::ceil_div(KV, 256), (unsigned)(batch * a.heads)),
                     dim3(64), 0, st, c.states, a.factors, c.carry, KV, a.segments - 1);
}

// Outputs too large for the caches to hold for what reads them next are
// streamed: in whole rows past the caches, which keep the operands that other
// workgroups read again.  Measured, bf16: 134 MB (64 x 2048 steps, 8 heads of
// 64) 176 -> 164 us, 67 MB 109 -> 98; both passes of 128 x 1000 steps, 8 heads of
// 64, 493 -> 469 us, of 8 x 4096 steps, 16 heads of 128, 685 -> 672, 65536 steps of
// those 414 -> 407.  (With products of one piece and a product that reads the
// outputs next: 134 MB 224 -> 215 us, 67 MB 118 -> 115, 33 MB 69 -> 70, and 56 ->
// 55 alone.  Whole rows through the caches gained half of that, and lost 2 %
// where outputs are small; 32 bytes of a row past the caches lost a quarter.)
void outputs_pass(hipStream_t st, int dtype, AttnArgs a, int batch) {
  const int D = padded(a.role[0].x.width, a.role[0].z.width);
  int64_t columns = 0;
  for (int i = 0; i < a.roles; ++i) columns += a.role[i].z.width;
  a.streamed = (int64_t)batch * a.steps * a.heads * columns * (dtype == ATTN_F32 ? 4 : 2) >= 64 << 20;
  const unsigned grid = (unsigned)((int64_t)batch * a.heads * a.segments * a.roles);
  if (dtype == ATTN_F32) launch_width<float, false>(st, a, D, grid);
  else launch_width<uint16_t, false>(st, a, D, grid);
}

// `least`: rows of sequences are read 16 bytes at a time.
int check_sizes(const char* what, int dtype, int batch, int steps, int heads, int kv_heads, int K, int V, int least) {
  if (dtype != ATTN_F32 && dtype != ATTN_BF16) return ppo::set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || heads < 0 || kv_heads < 0)
    return ppo::set_error(PPO_ERR_ARG, "%s: negative size (batch %d steps %d heads %d, %d)", what, batch, steps, heads,
                          kv_heads);
  if (K > MAX_WIDTH || V > MAX_WIDTH || K < least || V < least)
    return ppo::set_error(PPO_ERR_ARG, "%s: widths %d, %d outside %d .. %d", what, K, V, least, MAX_WIDTH);
  if (heads > 0 && (kv_heads == 0 || heads % kv_heads))
    return ppo::set_error(PPO_ERR_ARG, "%s: %d heads do not share %d key heads evenly", what, heads, kv_heads);
  if (heads > (1 << 23) / MAX_WIDTH)  // an output step's elements, as check_strides
    return ppo::set_error(PPO_ERR_ARG, "%s: %d heads above %d", what, heads, (1 << 23) / MAX_WIDTH);
  // a launch's threads (three outputs of the backward pass, 512 each; two slices of a step, 256 each) are
  // counted in 32 bits
  const int64_t most = least > 1 ? 1 << 21 : (1 << 23) - 1;
  if ((int64_t)batch * heads > most)
    return ppo::set_error(PPO_ERR_ARG, "%s: batch x heads above %lld", what, (long long)most);
  if (steps > 1 << 30) return ppo::set_error(PPO_ERR_ARG, "%s: %d steps above 2^30", what, steps);
  return PPO_OK;
}

bool empty(int batch, int heads) { return batch == 0 || heads == 0; }

// A lane's byte within a chunk is counted in 32 bits.  (One step has no stride.)
int check_strides(const char* what, const int64_t* strides, int operands, int steps) {
  for (int i = 0; i < operands; ++i) {
    const int64_t st = strides[3 * i + 1];
    if (steps > 1 && (st < 0 || st > 1 << 23))
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

PPO_EXPORT int ppo_linear_attention_min_width(int dtype) { return dtype == ATTN_BF16 ? 8 : 4; }

PPO_EXPORT size_t ppo_linear_attention_workspace(int dtype, int batch, int steps, int heads, int key_width,
                                                 int value_width) {
  if (check_sizes("ppo_linear_attention_workspace", dtype, batch, steps, heads, heads, key_width, value_width, 1))
    return 0;
  if (empty(batch, heads)) return 0;
  return sizeof(float) * (size_t)state_floats(dtype, batch, steps, heads, key_width, value_width);
}

PPO_EXPORT size_t ppo_linear_attention_bwd_workspace(int dtype, int batch, int steps, int heads, int kv_heads,
                                                     int key_width, int value_width) {
  if (check_sizes("ppo_linear_attention_bwd_workspace", dtype, batch, steps, heads, kv_heads, key_width, value_width,
                  1))
    return 0;
  if (empty(batch, heads)) return 0;
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
  if (int rc = check_sizes(what, dtype, batch, steps, heads, kv_heads, K, V, ppo_linear_attention_min_width(dtype))) return rc;
  if (empty(batch, heads)) return PPO_OK;
  if (!log_decay || !final || !strides || (steps > 0 && (!q || !k || !v || !out)))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 3, steps)) return rc;
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
  if (int rc = check_sizes(what, dtype, batch, steps, heads, kv_heads, K, V, ppo_linear_attention_min_width(dtype))) return rc;
  if (empty(batch, heads)) return PPO_OK;
  if (!log_decay || !strides || (steps > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv)))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  if (int rc = check_strides(what, strides, 4, steps)) return rc;
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
      const dim3 grid((unsigned)std::min<int64_t>(1 << 16, ppo::ceil_div64(n, 256)));
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
  if (int rc = check_sizes(what, dtype, batch, 1, heads, kv_heads, K, V, 1)) return rc;
  if (empty(batch, heads)) return PPO_OK;
  if (!q || !k || !v || !strides || !log_decay || !carry || !final || !out)
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  StepArgs a{q, k, v, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], log_decay, done, carry,
             final, out, scale, heads, heads / kv_heads, K, V, 0, 0};
  // a workgroup a head, or slices of at least 32 columns where those are too
  // few to fill the chip (float32 heads of 128 whole / in slices of 32: 32 of
  // them 6.6 / 4.2 us, 128 of them 7.5 / 5.5, 2048 of them 46.4 / 49.1)
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
