// The norms after and before a block, with the block's gate, the residual
// scale and the sum into the residual stream in the same pass, and its
// vector-Jacobian product.
//
// Per row of D columns (one step of one sequence), u the block's output, x the
// residual stream:
//   n = u / sqrt(mean(u^2) + eps) * post     (or n = u: no norm of the block's output)
//   y = x + scale * gate * n                 (gate: 1, g, or sigmoid(g))
//   z = y / sqrt(mean(y^2) + eps) * pre
// y is the new stream, z what the next block reads, both from the unrounded y.
// Backward, from the cotangents dy and dz, with u' = u ru and y' = y ry (ru, ry
// the two rows' 1 / rms, kept by the forward), q = scale gate:
//   e = dz pre, m = mean(e y'), dx = dy + ry (e - y' m),
//   dgate = dx scale n, f = dx q post, du = ru (f - u' mean(f u')),
//   dpre = sum dz y', dscale = sum dx gate n, dpost = sum dx q u'.
// mean(f u') is linear in m, so that one exchange of three sums serves both:
//   mean(f u') = mean((dy + ry e) q post u') - m mean(ry y' q post u').
//
// scale and post enter y, dx and du as their product alone, and both their
// gradients are one sum: with s = sum dx gate u', dscale = post s, dpost = scale s.
//
// A thread holds 8 columns of a row and their scales for all its rows; a row is
// L lanes of a wave (up to 512 columns) or one workgroup, and the next row's
// operands are on their way while one is formed.  Sums are float32, the
// lanes' by butterflies, the waves' in order.
//
// What bounds it is HBM: 65536 rows of 2048 bf16 columns with a float32 stream 322 us
// (5.0 TB/s); 128000 of 640 bf16 with gates 174 us, backward 277 (4.7 TB/s both) and
// 7 for the scales; 15984 of 1333 float32 101 and 153 us (4.2, 4.5 TB/s).  64 rows of
// 1000 take 4.5 us: a launch, and a row's two sums one after the other.
#include "row_io.h"

#include <algorithm>

namespace {

using namespace ppo;

enum NormDtype { NORM_F32 = 0, NORM_BF16 = 1 };

constexpr int THREADS = 256;               // of a workgroup of narrow rows, and of most wide ones
constexpr int MAX_THREADS = 1024;
constexpr int NARROW = 64 * UNIT;          // widest row of one wave's lanes
constexpr int MAX_WIDTH = MAX_THREADS * UNIT;
// Workgroups a CU, of `waves` waves each: whole numbers, or some CUs hold one more than others and the launch takes as
// long as they do (67M elements, both passes, for as many waves spread unevenly: rows of 3000 bf16 columns 375 us for 456,
// 8192 381 for 469, 8192 float32 781 for 1079; forward alone, 134M, 5632 bf16 275 for 331, 8192 float32 511 for 613).
constexpr int CUS = 256;
// Forward at most 24 waves (rows of 2304 bf16 columns, five waves: 286 us, with 25 309).
int fwd_groups(int waves) { return std::max(1, 24 / waves); }
// Backward at least 8, and 12 for narrow bf16 rows: those whose last lanes are idle have too little on its way with 8
// (both passes, 67M elements: rows of 40 385 us for 428, 136 429 for 489, 300 422 for 469, 640 386 for 405, 768 370 for 371;
// but full ones lose, of 16 to 512 columns 1 to 3 %, and wider ones, 700 413 for 403, 800 392 for 374, 1024 368 for 353).
int bwd_groups(int dtype, int D, int waves) { return ceil_div(dtype == NORM_BF16 && D <= 768 ? 12 : 8, waves); }

enum Gate { GATE_NONE, GATE_PLAIN, GATE_SIGMOID };

struct ResidualArgs {
  const void* block;
  const void* gate;       // or null
  const void* residual;
  const float* post;      // scales [D], or null (ones)
  const float* scale;
  const float* pre;
  void* stream;           // forward
  void* normed;
  float* stats;           // [rows, 2]: ru, ry (forward: or null)
  const void* dstream;    // backward, each or null (zeros)
  const void* dnormed;
  void* dblock;
  void* dgate;            // or null
  void* dresidual;
  float* partials;        // [workgroups, 2, D]: sum dx gate u', dpre
  RowStride block_s, gate_s, residual_s, dstream_s, dnormed_s;
  Divisor steps;
  uint32_t rows;
  int D, lanes_log2;
  float eps;
  bool post_norm;
};

// Sums over a row: its lanes (narrow), or the workgroup, whose waves' sums
// meet in LDS.  `slot`: another at each call until every wave has passed a
// later one.
template <bool WIDE, int N> struct RowSum {
  float (*waves)[MAX_THREADS / 64][N];
  int log2;
  __device__ __forceinline__ void operator()(float (&v)[N], int slot) const {
    if constexpr (!WIDE) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i], log2);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = wave_sum_lanes(v[i]);
      const int wave = threadIdx.x >> 6, count = blockDim.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) waves[slot][wave][i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.f;
      for (int w = 0; w < count; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += waves[slot][w][i];
    }
  }
};

// Which rows and columns a thread takes.  The last columns of a row that 8 does
// not divide are the row's last 8, some of them another thread's too: those
// (j < skip), and all of a thread past the row's end, count in no sum over the row.
struct Place {
  uint32_t row, step;  // its first row, and from one to its next
  int col, skip;
  bool stores;
};
template <bool WIDE> __device__ __forceinline__ Place place_of(const ResidualArgs& p) {
  Place r;
  int col;
  if constexpr (WIDE) {
    r.row = blockIdx.x;
    r.step = gridDim.x;
    col = threadIdx.x * UNIT;
  } else {
    const int L = 1 << p.lanes_log2;
    r.row = (blockIdx.x * THREADS + threadIdx.x) >> p.lanes_log2;
    r.step = (gridDim.x * THREADS) >> p.lanes_log2;
    col = (threadIdx.x & (L - 1)) * UNIT;
  }
  r.col = max(0, min(col, p.D - UNIT));
  r.skip = col - r.col;
  r.stores = col < p.D;
  return r;
}
// A unit of a row; of rows of fewer than 8 columns what there is of it.
template <typename S> __device__ __forceinline__ void load_part(const S* p, int D, Unit8<S>& u) {
  if (D >= UNIT) __builtin_memcpy(u.w, p, sizeof(u.w));
  else load_unit(p, D, u);
}
template <typename S> __device__ __forceinline__ void store_part(S* p, int D, const float (&v)[UNIT]) {
  store_unit(p, min(D, UNIT), v);
}
__device__ __forceinline__ float scale_of(const float* p, int col, int D) { return p && col < D ? p[col] : 1.f; }

template <typename T, typename R> struct Loaded {
  Unit8<T> u, g, dz;
  Unit8<R> x, dy;
  float ru, ry;
};

template <int GATE, bool BWD, typename T, typename R>
__device__ __forceinline__ void load(const ResidualArgs& p, uint32_t row, const Place& at, Loaded<T, R>& v) {
  load_part(static_cast<const T*>(p.block) + row_offset(row, p.steps, p.block_s) + at.col, p.D, v.u);
  load_part(static_cast<const R*>(p.residual) + row_offset(row, p.steps, p.residual_s) + at.col, p.D, v.x);
  if constexpr (GATE != GATE_NONE)
    load_part(static_cast<const T*>(p.gate) + row_offset(row, p.steps, p.gate_s) + at.col, p.D, v.g);
  if constexpr (BWD) {
    // (a cotangent that is not there: the operand in its place, and zeros selected for it)
    load_part(static_cast<const T*>(p.dnormed) + row_offset(row, p.steps, p.dnormed_s) + at.col, p.D, v.dz);
    load_part(static_cast<const R*>(p.dstream) + row_offset(row, p.steps, p.dstream_s) + at.col, p.D, v.dy);
    v.ru = p.stats[2 * (int64_t)row];
    v.ry = p.stats[2 * (int64_t)row + 1];
  }
}
// The gate and (sigmoid) its slope.
template <int GATE, typename T> __device__ __forceinline__ float gate_of(const Unit8<T>& g, int j, float& slope) {
  slope = 1.f;
  if constexpr (GATE == GATE_NONE) return 1.f;
  else if constexpr (GATE == GATE_PLAIN) return value(g, j);
  else {
    float rest;
    const float s = sigmoid(value(g, j), rest);
    slope = s * rest;
    return s;
  }
}

template <typename T, typename R, int GATE, bool WIDE, int MOST>
__global__ void __launch_bounds__(MOST) residual_norm_fwd_kernel(ResidualArgs p) {
  __shared__ float waves[2][MAX_THREADS / 64][1];
  const RowSum<WIDE, 1> row_sum{waves, p.lanes_log2};
  const Place at = place_of<WIDE>(p);
  float mix[UNIT], pre[UNIT];   // mix: post scale
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    mix[j] = scale_of(p.post, at.col + j, p.D) * scale_of(p.scale, at.col + j, p.D);
    pre[j] = scale_of(p.pre, at.col + j, p.D);
  }
  const float over_d = 1.f / (float)p.D;
  int slot = 0;
  Loaded<T, R> next;
  load<GATE, false>(p, min(at.row, p.rows - 1), at, next);
  for (uint32_t row = at.row; __any(row < p.rows); row += at.step) {   // (a wave's rows end together)
    const Loaded<T, R> v = next;
    load<GATE, false>(p, min(row + at.step, p.rows - 1), at, next);
    float y[UNIT], ru = 1.f, sum[1];
    if (p.post_norm) {
      sum[0] = 0.f;
#pragma unroll
      for (int j = 0; j < UNIT; ++j) {
        const float u = j >= at.skip ? value(v.u, j) : 0.f;
        sum[0] = __fmaf_rn(u, u, sum[0]);
      }
      row_sum(sum, slot);
      slot ^= 1;
      ru = rsqrtf(__fmaf_rn(sum[0], over_d, p.eps));
    }
    sum[0] = 0.f;
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      float slope;
      y[j] = __fmaf_rn(mix[j], gate_of<GATE>(v.g, j, slope) * (value(v.u, j) * ru), value(v.x, j));
      const float counted = j >= at.skip ? y[j] : 0.f;
      sum[0] = __fmaf_rn(counted, counted, sum[0]);
    }
    row_sum(sum, slot);
    slot ^= 1;
    const float ry = rsqrtf(__fmaf_rn(sum[0], over_d, p.eps));
    if (row >= p.rows || !at.stores) continue;
    const int64_t out = (int64_t)row * p.D + at.col;
    store_part(static_cast<R*>(p.stream) + out, p.D, y);
#pragma unroll
    for (int j = 0; j < UNIT; ++j) y[j] = y[j] * ry * pre[j];
    store_part(static_cast<T*>(p.normed) + out, p.D, y);
    if (p.stats && at.col + at.skip == 0) {
      p.stats[2 * (int64_t)row] = ru;
      p.stats[2 * (int64_t)row + 1] = ry;
    }
  }
}

template <typename T, typename R, int GATE, bool WIDE, int MOST>
__global__ void __launch_bounds__(MOST) residual_norm_bwd_kernel(ResidualArgs p, bool has_dstream, bool has_dnormed) {
  __shared__ float waves[2][MAX_THREADS / 64][3];
  const RowSum<WIDE, 3> row_sum{waves, p.lanes_log2};
  const Place at = place_of<WIDE>(p);
  float mix[UNIT], pre[UNIT], dmix[UNIT], dpre[UNIT];
#pragma unroll
  for (int j = 0; j < UNIT; ++j) {
    mix[j] = scale_of(p.post, at.col + j, p.D) * scale_of(p.scale, at.col + j, p.D);
    pre[j] = scale_of(p.pre, at.col + j, p.D);
    dmix[j] = dpre[j] = 0.f;
  }
  const float over_d = 1.f / (float)p.D;
  int slot = 0;
  // (9 to 16 waves leave no registers for a next row: 67M elements in rows of 8192 bf16 columns, both passes, 358 us for 432)
  constexpr bool AHEAD = MOST <= 512;
  Loaded<T, R> next;
  if constexpr (AHEAD) load<GATE, true>(p, min(at.row, p.rows - 1), at, next);
  for (uint32_t row = at.row; __any(row < p.rows); row += at.step) {
    if constexpr (!AHEAD) load<GATE, true>(p, min(row, p.rows - 1), at, next);
    const Loaded<T, R> v = next;
    if constexpr (AHEAD) load<GATE, true>(p, min(row + at.step, p.rows - 1), at, next);
    const bool live = row < p.rows;
    const float ru = v.ru, ry = v.ry;
    // un = u', gun = gate u', yn = y'
    float un[UNIT], gun[UNIT], yn[UNIT], dx[UNIT], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      float slope;
      un[j] = value(v.u, j) * ru;
      gun[j] = gate_of<GATE>(v.g, j, slope) * un[j];
      yn[j] = __fmaf_rn(mix[j], gun[j], value(v.x, j)) * ry;
      const float dz = has_dnormed ? value(v.dz, j) : 0.f, e = dz * pre[j];
      if (WIDE || live) dpre[j] = __fmaf_rn(dz, yn[j], dpre[j]);
      dx[j] = __fmaf_rn(ry, e, has_dstream ? value(v.dy, j) : 0.f);
      const float k = j >= at.skip ? mix[j] * gun[j] : 0.f;
      sum[0] = __fmaf_rn(j >= at.skip ? e : 0.f, yn[j], sum[0]);
      sum[1] = __fmaf_rn(dx[j], k, sum[1]);
      sum[2] = __fmaf_rn(yn[j], k, sum[2]);
    }
    row_sum(sum, slot);
    slot ^= 1;
    const float m = sum[0] * over_d * ry;
    const float mu = p.post_norm ? __fmaf_rn(-m, sum[2], sum[1]) * over_d : 0.f;
    float du[UNIT], dg[UNIT];
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      float slope;
      const float gate = gate_of<GATE>(v.g, j, slope);
      dx[j] = __fmaf_rn(-yn[j], m, dx[j]);
      if (WIDE || live) dmix[j] = __fmaf_rn(dx[j], gun[j], dmix[j]);
      const float dn = dx[j] * mix[j];
      dg[j] = dn * un[j] * slope;
      du[j] = ru * __fmaf_rn(-un[j], mu, dn * gate);
    }
    if (!live || !at.stores) continue;
    const int64_t out = (int64_t)row * p.D + at.col;
    store_part(static_cast<R*>(p.dresidual) + out, p.D, dx);
    store_part(static_cast<T*>(p.dblock) + out, p.D, du);
    if constexpr (GATE != GATE_NONE) {
      if (p.dgate) store_part(static_cast<T*>(p.dgate) + out, p.D, dg);
    }
  }
  if (!p.partials) return;
  float* mine = p.partials + (int64_t)blockIdx.x * 2 * p.D;
  if constexpr (WIDE) {
    if (!at.stores) return;
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      mine[at.col + j] = dmix[j];
      mine[p.D + at.col + j] = dpre[j];
    }
  } else {
    // the rows of the workgroup side by side, added in their order
    __shared__ float sums[THREADS * UNIT];
    const int L = 1 << p.lanes_log2;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < UNIT; ++j) sums[j * THREADS + threadIdx.x] = w == 0 ? dmix[j] : dpre[j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.D; c += THREADS) {
        const int lane = c / UNIT, place = c - max(0, min(lane * UNIT, p.D - UNIT));
        float s = 0.f;
        for (int g = lane; g < THREADS; g += L) s += sums[place * THREADS + g];
        mine[w * p.D + c] = s;
      }
    }
  }
}

// The scales' gradients from the workgroups' sums: 16 columns a workgroup, 64
// shares of the sums, each in their order, then the shares' by a tree.
constexpr int SUM_COLUMNS = 16, SUM_SHARES = 64;
__global__ void __launch_bounds__(SUM_COLUMNS* SUM_SHARES)
    residual_norm_scale_kernel(const float* partials, int blocks, int D, const float* post, const float* scale,
                               float* dpost, float* dscale, float* dpre) {
  __shared__ float sums[SUM_SHARES][SUM_COLUMNS];
  const int c = threadIdx.x % SUM_COLUMNS, share = threadIdx.x / SUM_COLUMNS, i = blockIdx.x * SUM_COLUMNS + c;
  const int each = (blocks + SUM_SHARES - 1) / SUM_SHARES, b1 = min(blocks, (share + 1) * each);
  float s = 0.f;
  if (i < 2 * D) {
    for (int b0 = share * each; b0 < b1; b0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = partials[(int64_t)min(b0 + k, b1 - 1) * 2 * D + i];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += b0 + k < b1 ? v[k] : 0.f;
    }
  }
  sums[share][c] = s;
  for (int half = SUM_SHARES / 2; half > 0; half /= 2) {
    __syncthreads();
    if (share < half) sums[share][c] += sums[share + half][c];
  }
  if (share > 0 || i >= 2 * D) return;
  s = sums[0][c];
  if (i >= D) {
    if (dpre) dpre[i - D] = s;
  } else {
    if (dpost) dpost[i] = scale ? scale[i] * s : s;
    if (dscale) dscale[i] = post ? post[i] * s : s;
  }
}

// ---- launches
int lanes_log2_of(int D) {
  int log2 = 0;
  while ((UNIT << log2) < D) ++log2;
  return log2;
}

// Threads and workgroups of a launch.
struct Shape {
  bool wide;
  unsigned threads, blocks;
};
Shape shape_of(int64_t rows, int D, int dtype, bool backward) {
  Shape s;
  s.wide = D > NARROW;
  s.threads = s.wide ? (unsigned)(64 * ceil_div(D, NARROW)) : THREADS;
  const int64_t at_once = s.wide ? 1 : THREADS >> lanes_log2_of(D);
  const int waves = (int)s.threads / 64, groups = backward ? bwd_groups(dtype, D, waves) : fwd_groups(waves);
  s.blocks = (unsigned)std::min<int64_t>(CUS * groups, ceil_div64(rows, at_once));
  return s;
}

int check(const char* what, int dtype, int stream_dtype, int batch, int steps, int width) {
  if ((dtype != NORM_F32 && dtype != NORM_BF16) || (stream_dtype != NORM_F32 && stream_dtype != dtype))
    return set_error(PPO_ERR_ARG, "%s: bad dtype %d, stream %d", what, dtype, stream_dtype);
  if (batch < 0 || steps < 0 || width < 0)
    return set_error(PPO_ERR_ARG, "%s: bad size (batch %d steps %d width %d)", what, batch, steps, width);
  if (width > MAX_WIDTH) return set_error(PPO_ERR_ARG, "%s: width %d above %d", what, width, MAX_WIDTH);
  if ((int64_t)batch * steps > INT32_MAX - (1 << 20))
    return set_error(PPO_ERR_ARG, "%s: batch x steps above 2^31 - 2^20 - 1", what);
  return PPO_OK;
}

ResidualArgs common_args(const void* block, const void* gate, const void* residual, const int64_t* strides,
                         const float* post, const float* scale, const float* pre, int post_norm, float epsilon, int batch,
                         int steps, int width) {
  ResidualArgs a{};
  a.block = block;
  a.gate = gate;
  a.residual = residual;
  a.post = post;
  a.scale = scale;
  a.pre = pre;
  a.block_s = RowStride{strides[0], strides[1]};
  a.residual_s = RowStride{strides[2], strides[3]};
  a.gate_s = RowStride{strides[4], strides[5]};
  a.steps = divisor((uint32_t)steps);
  a.rows = (uint32_t)((int64_t)batch * steps);
  a.D = width;
  a.lanes_log2 = width <= NARROW ? lanes_log2_of(width) : 0;
  a.eps = epsilon;
  a.post_norm = post_norm != 0;
  return a;
}

template <typename T, typename R, int GATE, bool WIDE, int MOST>
void launch_shape(hipStream_t st, ResidualArgs a, const Shape& s, bool backward) {
  const dim3 g(s.blocks), t(s.threads);
  if (backward) {
    const bool dstream = a.dstream, dnormed = a.dnormed;
    if (!dstream) {
      a.dstream = a.residual;
      a.dstream_s = a.residual_s;
    }
    if (!dnormed) {
      a.dnormed = a.block;
      a.dnormed_s = a.block_s;
    }
    hipLaunchKernelGGL((residual_norm_bwd_kernel<T, R, GATE, WIDE, MOST>), g, t, 0, st, a, dstream, dnormed);
  } else {
    hipLaunchKernelGGL((residual_norm_fwd_kernel<T, R, GATE, WIDE, MOST>), g, t, 0, st, a);
  }
}
template <typename T, typename R, int GATE>
void launch_gate(hipStream_t st, const ResidualArgs& a, const Shape& s, bool backward) {
  if (!s.wide) launch_shape<T, R, GATE, false, THREADS>(st, a, s, backward);
  else if (s.threads <= THREADS) launch_shape<T, R, GATE, true, THREADS>(st, a, s, backward);
  else if (s.threads <= 512) launch_shape<T, R, GATE, true, 512>(st, a, s, backward);
  else launch_shape<T, R, GATE, true, MAX_THREADS>(st, a, s, backward);
}
template <typename T, typename R>
void launch(hipStream_t st, const ResidualArgs& a, const Shape& s, int gate_sigmoid, bool backward) {
  if (!a.gate) launch_gate<T, R, GATE_NONE>(st, a, s, backward);
  else if (gate_sigmoid) launch_gate<T, R, GATE_SIGMOID>(st, a, s, backward);
  else launch_gate<T, R, GATE_PLAIN>(st, a, s, backward);
}
void launch_typed(hipStream_t st, const ResidualArgs& a, const Shape& s, int gate_sigmoid, bool backward, int dtype,
                  int stream_dtype) {
  if (dtype == NORM_F32) launch<float, float>(st, a, s, gate_sigmoid, backward);
  else if (stream_dtype == NORM_F32) launch<uint16_t, float>(st, a, s, gate_sigmoid, backward);
  else launch<uint16_t, uint16_t>(st, a, s, gate_sigmoid, backward);
}

}  // namespace

PPO_EXPORT int ppo_residual_norm_max_width(void) { return MAX_WIDTH; }

PPO_EXPORT int ppo_residual_norm_fwd(void* stream, int dtype, int stream_dtype, const void* block,
                                     const void* residual, const void* gate, const int64_t* strides,
                                     const float* post_scale, const float* residual_scale, const float* pre_scale,
                                     int post_norm, int gate_sigmoid, float epsilon, void* stream_out, void* normed,
                                     float* stats, int batch, int steps, int width) {
  const char* what = "ppo_residual_norm_fwd";
  if (int rc = check(what, dtype, stream_dtype, batch, steps, width)) return rc;
  if ((int64_t)batch * steps == 0 || width == 0) return PPO_OK;
  if (!block || !residual || !strides || !stream_out || !normed) return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  ResidualArgs a = common_args(block, gate, residual, strides, post_scale, residual_scale, pre_scale, post_norm,
                               epsilon, batch, steps, width);
  a.stream = stream_out;
  a.normed = normed;
  a.stats = stats;
  launch_typed(as_stream(stream), a, shape_of(a.rows, width, dtype, false), gate_sigmoid, false, dtype, stream_dtype);
  return check_launch(what);
}

PPO_EXPORT size_t ppo_residual_norm_bwd_workspace(int dtype, int batch, int steps, int width) {
  if (batch <= 0 || steps <= 0 || width <= 0 || width > MAX_WIDTH) return 0;
  return sizeof(float) * 2 * (size_t)width * shape_of((int64_t)batch * steps, width, dtype, true).blocks;
}

PPO_EXPORT int ppo_residual_norm_bwd(void* stream, int dtype, int stream_dtype, const void* block,
                                     const void* residual, const void* gate, const void* dstream,
                                     const void* dnormed, const int64_t* strides, const float* post_scale,
                                     const float* residual_scale, const float* pre_scale, int post_norm,
                                     int gate_sigmoid, const float* stats, void* dblock, void* dresidual, void* dgate,
                                     float* dpost_scale, float* dresidual_scale, float* dpre_scale, void* workspace,
                                     size_t workspace_bytes, int batch, int steps, int width) {
  const char* what = "ppo_residual_norm_bwd";
  if (int rc = check(what, dtype, stream_dtype, batch, steps, width)) return rc;
  if (width == 0) return PPO_OK;
  const bool none = (int64_t)batch * steps == 0, scales = dpost_scale || dresidual_scale || dpre_scale;
  if (!none && (!block || !residual || !strides || !stats || !dblock || !dresidual))
    return set_error(PPO_ERR_ARG, "%s: null buffer", what);
  const size_t need = scales ? ppo_residual_norm_bwd_workspace(dtype, batch, steps, width) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  unsigned blocks = 0;
  if (!none) {
    ResidualArgs a = common_args(block, gate, residual, strides, post_scale, residual_scale, pre_scale, post_norm,
                                 0.f, batch, steps, width);
    a.stats = const_cast<float*>(stats);
    a.dstream = dstream;
    a.dnormed = dnormed;
    a.dstream_s = RowStride{strides[6], strides[7]};
    a.dnormed_s = RowStride{strides[8], strides[9]};
    a.dblock = dblock;
    a.dgate = gate ? dgate : nullptr;
    a.dresidual = dresidual;
    a.partials = scales ? static_cast<float*>(workspace) : nullptr;
    const Shape s = shape_of(a.rows, width, dtype, true);
    blocks = s.blocks;
    launch_typed(as_stream(stream), a, s, gate_sigmoid, true, dtype, stream_dtype);
  }
  if (scales)
    hipLaunchKernelGGL(residual_norm_scale_kernel, dim3((unsigned)ceil_div(2 * width, SUM_COLUMNS)),
                       dim3(SUM_COLUMNS * SUM_SHARES), 0,
                       as_stream(stream), static_cast<const float*>(workspace), (int)blocks, width, post_scale,
                       residual_scale, dpost_scale, dresidual_scale, dpre_scale);
  return check_launch(what);
}
