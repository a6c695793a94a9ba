// Norms of queries and keys for each head, with the position rotation in the
// same pass, and its vector-Jacobian product.
//
// Per row x of D columns (one head of one step) at position p:
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r scale
//   out = y with each pair (y_a, y_b) of frequency f turned by the angle p f:
//     (y_a cos - y_b sin, y_b cos + y_a sin); the pairs are columns (i, i + P)
//     or, interleaved, (2 i, 2 i + 1), i < P; columns past 2 P stay as they are.
// Backward, from the cotangent c of out: e = c turned back, dscale += e x r,
//   dx = r (e scale - x r^2 mean(e scale x)).
//
// A wave takes a tile of steps with all heads of both: the angles' sines and
// cosines are formed once a step and pair (p f in float64, since float32 is off
// by up to p 2^-24 radians, and its turns brought within an eighth before the
// float32 series) and read from LDS by every head, and the next tile's rows are
// on their way while this one's are finished.  L lanes hold a row, each in units
// of two chunks of VW columns that hold whole pairs, so the rotation needs no
// lane exchange; the sums over a row are L-lane butterflies in float32.  Waves
// share nothing but the scales and frequencies, so none waits for another.
// Bound by HBM: x is read and out written once, at
// 5.4 TB/s forward (65536 steps, 16 heads of 128, bf16: 200 us) and 4.9 TB/s
// backward (128 x 1000 steps, 8 heads of 64, bf16: 162 us).
#include "split_f32.h"

#include <algorithm>

namespace {

enum NormDtype { NORM_F32 = 0, NORM_BF16 = 1 };

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MAX_DIM = 256;
constexpr int MAX_COLUMNS = MAX_DIM + 64;  // with those of a row's last lane past its end
constexpr int TILE_ANGLES = 512;  // most angles of a wave's tile
constexpr int TILE_STEPS = 64;    // and steps: a lane each
// Rows a lane group has in flight of each part, and most workgroups (the
// backward's leave a partial sum of dscale each).  Measured, bf16, 128 x 1000
// steps, 8 heads of 64 of both: backward 162 us, with half and twice as many
// workgroups 180 and 172, with two rows (which leave two workgroups a CU for
// three) 187; forward of 65536 steps, 16 heads of 128: 200 us, with one row 209.
constexpr int FWD_ROWS = 2, BWD_ROWS = 1;
constexpr int FWD_BLOCKS = 4096, BWD_BLOCKS = 768;

struct Rows {
  const void* x;
  const void* cot;      // backward
  const float* scale;   // [D], or null (ones)
  void* out;            // [tokens, heads, D]
  int64_t sb, st, sh;   // element strides of x
  int64_t cb, ct, ch;   // and of cot
  int heads;
  uint32_t inverse;     // 2^32 / heads, rounded up
};

struct NormArgs {
  Rows part[2];         // queries, keys
  const double* frequencies;
  const int32_t* positions;  // [batch, steps], or null (the step itself)
  float* partials;      // backward: [workgroups, 2, D]
  float eps;
  uint32_t tokens, steps, inverse_steps, inverse_pairs;  // inverses: 2^32 / x, rounded up
  int D, P, tile, lanes_log2;
};

// A chunk of VW columns as loaded (words of 4 bytes, or one element of 2).
template <typename T, int VW> struct Raw {
  static constexpr int WORDS = VW * (int)sizeof(T) < 4 ? 1 : VW * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
};
template <int VW> __device__ __forceinline__ void load_row(const uint16_t* p, int left, Raw<uint16_t, VW>& v) {
  if (left >= VW) {
    if constexpr (VW == 1) v.w[0] = p[0];
    else __builtin_memcpy(v.w, p, 2 * VW);
  } else {
#pragma unroll
    for (int i = 0; i < Raw<uint16_t, VW>::WORDS; ++i) {
      const uint32_t lo = 2 * i < left ? p[2 * i] : 0, hi = 2 * i + 1 < left ? p[2 * i + 1] : 0;
      v.w[i] = lo | hi << 16;
    }
  }
}
template <int VW> __device__ __forceinline__ void load_row(const float* p, int left, Raw<float, VW>& v) {
  if (left >= VW) {
    __builtin_memcpy(v.w, p, 4 * VW);
  } else {
#pragma unroll
    for (int j = 0; j < VW; ++j) v.w[j] = j < left ? __float_as_uint(p[j]) : 0;
  }
}
template <int VW> __device__ __forceinline__ void widen(const Raw<uint16_t, VW>& r, float (&v)[VW]) {
#pragma unroll
  for (int j = 0; j < VW; ++j) v[j] = __uint_as_float(j & 1 ? r.w[j / 2] & 0xffff0000u : r.w[j / 2] << 16);
}
template <int VW> __device__ __forceinline__ void widen(const Raw<float, VW>& r, float (&v)[VW]) {
#pragma unroll
  for (int j = 0; j < VW; ++j) v[j] = __uint_as_float(r.w[j]);
}
template <int VW> __device__ __forceinline__ void store_row(uint16_t* p, int left, const float (&v)[VW]) {
  if constexpr (VW == 1) {
    if (left > 0) p[0] = (uint16_t)ppo::pack_bf16(v[0], v[0]);
  } else {
    uint32_t w[VW / 2];
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) w[j] = ppo::pack_bf16(v[2 * j], v[2 * j + 1]);
    if (left >= VW) {
      __builtin_memcpy(p, w, 2 * VW);
    } else {
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (j < left) p[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
  }
}
template <int VW> __device__ __forceinline__ void store_row(float* p, int left, const float (&v)[VW]) {
  if (left >= VW) {
    __builtin_memcpy(p, v, 4 * VW);
  } else {
#pragma unroll
    for (int j = 0; j < VW; ++j)
      if (j < left) p[j] = v[j];
  }
}

// Cosine and sine of `turns` whole turns (|turns| <= 1/2): the Taylor series
// about the nearest quarter turn, x within pi / 4; the terms left out are below
// x^11 / 11! < 2e-9.
__device__ __forceinline__ float2 cos_sin(float turns) {
  const float q = rintf(4.f * turns);
  const float x = __fmaf_rn(-0.25f, q, turns) * 6.283185307179586f, y = x * x;
  float s = __fmaf_rn(y, 1.f / 362880.f, -1.f / 5040.f);
  s = __fmaf_rn(y, s, 1.f / 120.f);
  s = __fmaf_rn(y, s, -1.f / 6.f);
  s = __fmaf_rn(x * y, s, x);
  float c = __fmaf_rn(y, -1.f / 3628800.f, 1.f / 40320.f);
  c = __fmaf_rn(y, c, -1.f / 720.f);
  c = __fmaf_rn(y, c, 1.f / 24.f);
  c = __fmaf_rn(y, c, -0.5f);
  c = __fmaf_rn(y, c, 1.f);
  const int k = (int)q & 3;   // the quarter
  const float cn = k & 1 ? s : c, sn = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -cn : cn, k >= 2 ? -sn : sn);
}

// Sum over the row's lanes (2^log2 of them, neighbours).
__device__ __forceinline__ float lanes_sum(float v, int log2) {
  if (log2 > 0) v += ppo::xor16<1>(v);
  if (log2 > 1) v += ppo::xor16<2>(v);
  if (log2 > 2) v += ppo::xor16<4>(v);
  if (log2 > 3) v += ppo::xor16<8>(v);
  if (log2 > 4) v = ppo::add_xor16(v);
  if (log2 > 5) v = ppo::add_xor32(v);
  return v;
}

// The columns of unit u of a row's `units`: chunks at a and b and the first
// pair of each (or -1: no rotation).  In the layout of halves the pairs'
// units come first, a chunk of first columns and that of their partners;
// otherwise chunks u and u + units, so that lanes read side by side.
struct Unit {
  int a, b, pair_a, pair_b;
};
template <int VW, bool INTER> __device__ __forceinline__ Unit unit_of(int u, int units, int P) {
  Unit r;
  const int rotated = INTER ? 0 : P / VW;
  if (u < rotated) {
    r.a = u * VW;
    r.b = P + r.a;
    r.pair_a = r.pair_b = r.a;
  } else {
    r.a = (INTER ? 0 : 2 * P) + (u - rotated) * VW;
    r.b = r.a + (units - rotated) * VW;
    r.pair_a = INTER && r.a < 2 * P ? r.a / 2 : -1;
    r.pair_b = INTER && r.b < 2 * P ? r.b / 2 : -1;
  }
  return r;
}

// The value, as if computed here: the LDS addresses that depend on it are
// formed for each row, where kept they would cost a wave's registers.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int VW>
__device__ __forceinline__ void load_scales(const float* scales, const Unit& u, float (&a)[VW], float (&b)[VW]) {
  // (a lane past the row's end multiplies zeros)
  const int at_a = here(min(u.a, MAX_COLUMNS - VW)), at_b = here(min(u.b, MAX_COLUMNS - VW));
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    a[j] = scales[at_a + j];
    b[j] = scales[at_b + j];
  }
}

// (a, b) turned by the unit's angles, back for `sign` -1.
template <int VW, bool INTER>
__device__ __forceinline__ void turn(float (&a)[VW], float (&b)[VW], const Unit& u, const float2* cs, int P,
                                     float sign) {
  if constexpr (INTER) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float(&v)[VW] = c ? b : a;
      const int first = here(c ? u.pair_b : u.pair_a);
      if (first < 0) continue;
#pragma unroll
      for (int j = 0; j < VW / 2; ++j) {
        const float2 w = cs[min(first + j, P - 1)];
        const float s = sign * w.y, x = v[2 * j], y = v[2 * j + 1];
        v[2 * j] = first + j < P ? x * w.x - y * s : x;
        v[2 * j + 1] = first + j < P ? y * w.x + x * s : y;
      }
    }
  } else if (u.pair_a >= 0) {
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      const float2 w = cs[u.pair_a + j];
      const float s = sign * w.y, x = a[j], y = b[j];
      a[j] = x * w.x - y * s;
      b[j] = y * w.x + x * s;
    }
  }
}

// A wave's own LDS accesses in order.
__device__ __forceinline__ void wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The rows of one lane group in flight: UNROLL of them, by the group's place.
template <typename T, int VW, int UPL, bool BWD> struct Batch {
  static constexpr int UNROLL = BWD ? BWD_ROWS : FWD_ROWS;
  Raw<T, VW> x[UNROLL][UPL][2];
  Raw<T, VW> c[BWD ? UNROLL : 1][UPL][2];
};

template <typename T, int VW, int UPL, bool INTER, bool BWD>
__global__ void __launch_bounds__(THREADS, BWD ? 3 : 2) qk_norm_kernel(NormArgs p) {
  __shared__ union {
    float2 angles[WAVES][TILE_ANGLES];
    float sums[BWD ? 2 * VW * UPL * THREADS : 1];
  } lds;
  __shared__ __attribute__((aligned(16))) float scales[2][MAX_COLUMNS];
  __shared__ double frequencies[MAX_DIM / 2];
  constexpr int UNROLL = Batch<T, VW, UPL, BWD>::UNROLL;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int L = 1 << p.lanes_log2, l = lane & (L - 1), D = p.D, P = p.P;
  const int group = lane >> p.lanes_log2, groups = 64 >> p.lanes_log2;
  float2* const cs = lds.angles[wave];
  const float over_d = 1.f / (float)D;
  Unit unit[UPL];
#pragma unroll
  for (int k = 0; k < UPL; ++k) unit[k] = unit_of<VW, INTER>(l + k * L, UPL * L, P);
  for (int i = tid; i < 2 * MAX_COLUMNS; i += THREADS) {
    const int w = i / MAX_COLUMNS, j = i % MAX_COLUMNS;
    scales[w][j] = p.part[w].scale && j < D ? p.part[w].scale[j] : 1.f;
  }
  for (int i = tid; i < P; i += THREADS) frequencies[i] = p.frequencies[i];
  float sum[2][UPL][2][VW];
  if constexpr (BWD) {
#pragma unroll
    for (int i = 0; i < 2 * UPL * 2 * VW; ++i) (&sum[0][0][0][0])[i] = 0.f;
  }
  __syncthreads();
  const uint32_t tiles = (p.tokens + p.tile - 1) / p.tile;
  // A tile: its first step (of all; its sequence and the step in that), its steps
  struct Tile {
    uint32_t t0, b0, s0;
    int n;
  };
  auto tile_at = [&](uint32_t tile) {
    Tile t;
    t.t0 = tile * p.tile;
    t.n = (int)min((uint32_t)p.tile, p.tokens - t.t0);
    t.b0 = t.t0 / p.steps;
    t.s0 = t.t0 - t.b0 * p.steps;
    return t;
  };
  auto step_of = [&](const Tile& tile, int s, uint32_t& b, uint32_t& t) {
    const uint32_t x = tile.s0 + s;
    const uint32_t wraps = p.steps > TILE_STEPS ? (x >= p.steps ? 1 : 0)
                           : p.steps > 1        ? __umulhi(x, p.inverse_steps)
                                                : x;
    b = tile.b0 + wraps;
    t = x - wraps * p.steps;
  };
  // row r of part w: step r / heads, head r % heads (exact: r heads < 2^32)
  auto place = [&](int w, int r, int& s, int& h) {
    s = p.part[w].heads == 1 ? r : (int)__umulhi((uint32_t)r, p.part[w].inverse);
    h = r - s * p.part[w].heads;
  };
  auto load = [&](const Tile& tile, int w, int r0, Batch<T, VW, UPL, BWD>& v) {
    const Rows& q = p.part[w];
    const int rows = tile.n * q.heads;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int r = r0 + u * groups;
      if (r < rows) {
        int s, h;
        place(w, r, s, h);
        uint32_t bb, tt;
        step_of(tile, s, bb, tt);
        const T* x = static_cast<const T*>(q.x) + ((int64_t)bb * q.sb + (int64_t)tt * q.st + (int64_t)h * q.sh);
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          load_row<VW>(x + unit[k].a, D - unit[k].a, v.x[u][k][0]);
          load_row<VW>(x + unit[k].b, D - unit[k].b, v.x[u][k][1]);
        }
        if constexpr (BWD) {
          const T* c = static_cast<const T*>(q.cot) + ((int64_t)bb * q.cb + (int64_t)tt * q.ct + (int64_t)h * q.ch);
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            load_row<VW>(c + unit[k].a, D - unit[k].a, v.c[u][k][0]);
            load_row<VW>(c + unit[k].b, D - unit[k].b, v.c[u][k][1]);
          }
        }
      }
    }
  };
  auto finish = [&](const Tile& tile, int w, int r0, const Batch<T, VW, UPL, BWD>& v) {
    const Rows& q = p.part[w];
    const int rows = tile.n * q.heads;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int r = r0 + u * groups;
      if (r >= rows) continue;
      int s, h;
      place(w, r, s, h);
      T* out = static_cast<T*>(q.out) + ((int64_t)(tile.t0 + s) * q.heads + h) * D;
      const float2* angles = cs + s * P;
      float a[UPL][VW], b[UPL][VW];
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < UPL; ++k) {
        widen(v.x[u][k][0], a[k]);
        widen(v.x[u][k][1], b[k]);
#pragma unroll
        for (int j = 0; j < VW; ++j) ss = __fmaf_rn(a[k][j], a[k][j], __fmaf_rn(b[k][j], b[k][j], ss));
      }
      ss = lanes_sum(ss, p.lanes_log2);
      const float rstd = rsqrtf(__fmaf_rn(ss, over_d, p.eps));
      if constexpr (!BWD) {
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          float wa[VW], wb[VW];
          load_scales(scales[w], unit[k], wa, wb);
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            a[k][j] = a[k][j] * rstd * wa[j];
            b[k][j] = b[k][j] * rstd * wb[j];
          }
          turn<VW, INTER>(a[k], b[k], unit[k], angles, P, 1.f);
          store_row<VW>(out + unit[k].a, D - unit[k].a, a[k]);
          store_row<VW>(out + unit[k].b, D - unit[k].b, b[k]);
        }
      } else {
        float ca[UPL][VW], cb[UPL][VW];
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          widen(v.c[u][k][0], ca[k]);
          widen(v.c[u][k][1], cb[k]);
          turn<VW, INTER>(ca[k], cb[k], unit[k], angles, P, -1.f);
          float wa[VW], wb[VW];
          load_scales(scales[w], unit[k], wa, wb);
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            a[k][j] *= rstd;
            b[k][j] *= rstd;
            sum[w][k][0][j] = __fmaf_rn(ca[k][j], a[k][j], sum[w][k][0][j]);
            sum[w][k][1][j] = __fmaf_rn(cb[k][j], b[k][j], sum[w][k][1][j]);
            ca[k][j] *= wa[j];
            cb[k][j] *= wb[j];
            m = __fmaf_rn(ca[k][j], a[k][j], __fmaf_rn(cb[k][j], b[k][j], m));
          }
        }
        m = lanes_sum(m, p.lanes_log2) * over_d;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            a[k][j] = rstd * __fmaf_rn(-a[k][j], m, ca[k][j]);
            b[k][j] = rstd * __fmaf_rn(-b[k][j], m, cb[k][j]);
          }
          store_row<VW>(out + unit[k].a, D - unit[k].a, a[k]);
          store_row<VW>(out + unit[k].b, D - unit[k].b, b[k]);
        }
      }
    }
  };
  auto position_of = [&](const Tile& tile) {  // of the lane's step
    return p.positions ? p.positions[tile.t0 + min(lane, tile.n - 1)] : 0;
  };
  Batch<T, VW, UPL, BWD> v[2];
  uint32_t index = blockIdx.x * WAVES + wave;
  Tile tile;
  int position = 0;
  if (index < tiles) {
    tile = tile_at(index);
    position = position_of(tile);
    load(tile, 0, group, v[0]);
    load(tile, 1, group, v[1]);
  }
  while (index < tiles) {
    for (int i0 = 0; i0 < tile.n * P; i0 += 64) {
      const int i = min(i0 + lane, tile.n * P - 1);
      const int s = P == 1 ? i : (int)__umulhi((uint32_t)i, p.inverse_pairs), f = i - s * P;
      uint32_t bb, tt;
      step_of(tile, s, bb, tt);
      const int at = __shfl(position, s);
      const double pos = p.positions ? (double)at : (double)tt;
      double turns = pos * frequencies[f] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      cs[i] = cos_sin((float)turns);
    }
    wave_lds();
    index += gridDim.x * WAVES;
    Tile next = tile;
    if (index < tiles) {
      next = tile_at(index);
      position = position_of(next);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      finish(tile, w, group, v[w]);
      for (int r0 = group + UNROLL * groups; r0 < tile.n * p.part[w].heads; r0 += UNROLL * groups) {
        load(tile, w, r0, v[w]);
        finish(tile, w, r0, v[w]);
      }
      if (index < tiles) load(next, w, group, v[w]);
    }
    wave_lds();
    tile = next;
  }
  if constexpr (BWD) {
    __syncthreads();
    // this workgroup's sums of dscale: a row group's lanes side by side, added
    // in the groups' order
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      constexpr int PER = 2 * VW * UPL;
#pragma unroll
      for (int k = 0; k < UPL; ++k)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          lds.sums[(k * 2 * VW + j) * THREADS + tid] = sum[w][k][0][j];
          lds.sums[(k * 2 * VW + VW + j) * THREADS + tid] = sum[w][k][1][j];
        }
      __syncthreads();
      for (int i = tid; i < PER * L; i += THREADS) {
        const int e = i >> p.lanes_log2, ll = i & (L - 1);
        float s = 0.f;
        for (int g = ll; g < THREADS; g += L) s += lds.sums[e * THREADS + g];
        const int k = e / (2 * VW), j = e % (2 * VW);
        const Unit u = unit_of<VW, INTER>(ll + k * L, UPL * L, P);
        const int col = j < VW ? u.a + j : u.b + j - VW;
        if (col < D) p.partials[((int64_t)blockIdx.x * 2 + w) * D + col] = s;
      }
      __syncthreads();
    }
  }
}

// dscale of both parts: the workgroups' sums, a column a wave, added in a fixed
// order (lane by lane, then the lanes' butterfly).
__global__ void __launch_bounds__(256) qk_norm_scale_kernel(const float* partials, int blocks, int D, float* dq_scale,
                                                            float* dk_scale) {
  const int lane = threadIdx.x & 63, col = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (col >= 2 * D) return;
  float s = 0.f;
  for (int b0 = lane; b0 < blocks; b0 += 64 * 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = partials[(int64_t)min(b0 + 64 * u, blocks - 1) * 2 * D + col];
#pragma unroll
    for (int u = 0; u < 8; ++u) s += b0 + 64 * u < blocks ? v[u] : 0.f;
  }
  s = ppo::wave_sum_lanes(s);
  float* out = col < D ? dq_scale : dk_scale;
  if (out && lane == 0) out[col < D ? col : col - D] = s;
}

// ---- launches
// Columns of a chunk: 16 bytes, or fewer where that does not divide the
// pairs of the layout of halves.
int chunk_columns(int dtype, int P, int interleaved) {
  int v = dtype == NORM_F32 ? 4 : 8;
  if (!interleaved)
    while (P % v) v /= 2;
  return v;
}

uint32_t inverse_of(int heads) { return heads > 1 ? (uint32_t)(((1ull << 32) + heads - 1) / heads) : 0; }

int lanes_log2_of(int D, int v) {
  int log2 = 0;
  while (log2 < 6 && (2 * v << log2) < D) ++log2;
  return log2;
}

// Steps of a wave's tile: rows of the part with fewer heads for every lane
// group's loads, no more angles than there is room for, a tile for every wave
// where there are few steps, and rows whose heads a 32-bit product tells.
int tile_of(int64_t tokens, int heads, int kv_heads, int pairs, int lanes_log2, int rows) {
  const int64_t most = std::max(heads, kv_heads), fewer = heads && kv_heads ? std::min(heads, kv_heads) : most;
  const int64_t busy = std::max<int64_t>(1, 64 * rows / (fewer << lanes_log2));
  return (int)std::max<int64_t>(1, std::min<int64_t>({busy, TILE_ANGLES / std::max(pairs, 1),
                                                      ppo::ceil_div64(tokens, 1024 * WAVES), TILE_STEPS,
                                                      (1ll << 32) / (most * most) - 1}));
}

unsigned blocks_of(int64_t tokens, int tile, int most) {
  return (unsigned)std::min<int64_t>(most, ppo::ceil_div64(tokens, (int64_t)tile * WAVES));
}

NormArgs common_args(float epsilon, int64_t tokens, int steps, int width, int pairs, int interleaved, int dtype,
                     int heads, int kv_heads, const double* frequencies, const int32_t* positions, int rows) {
  NormArgs a{};
  a.frequencies = frequencies;
  a.positions = positions;
  a.eps = epsilon;
  a.tokens = (uint32_t)tokens;
  a.steps = (uint32_t)steps;
  a.inverse_steps = inverse_of(steps);
  a.inverse_pairs = inverse_of(pairs);
  a.D = width;
  a.P = pairs;
  a.lanes_log2 = lanes_log2_of(width, chunk_columns(dtype, pairs, interleaved));
  a.tile = tile_of(tokens, heads, kv_heads, pairs, a.lanes_log2, rows);
  return a;
}

int check(const char* what, int dtype, int batch, int steps, int heads, int kv_heads, int dim, int pairs) {
  if (dtype != NORM_F32 && dtype != NORM_BF16) return ppo::set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || heads < 0 || kv_heads < 0 || dim < 0 || pairs < 0 || 2 * (int64_t)pairs > dim)
    return ppo::set_error(PPO_ERR_ARG, "%s: bad size (batch %d steps %d heads %d, %d width %d pairs %d)", what, batch,
                          steps, heads, kv_heads, dim, pairs);
  if (dim > MAX_DIM) return ppo::set_error(PPO_ERR_ARG, "%s: width %d above %d", what, dim, MAX_DIM);
  if (heads > 8192 || kv_heads > 8192)
    return ppo::set_error(PPO_ERR_ARG, "%s: %d, %d heads above 8192", what, heads, kv_heads);
  if ((int64_t)batch * steps > INT32_MAX) return ppo::set_error(PPO_ERR_ARG, "%s: batch x steps above 2^31 - 1", what);
  return PPO_OK;
}

template <typename T, bool BWD>
void launch_chunk(hipStream_t st, const NormArgs& a, int v, bool interleaved, unsigned grid) {
  constexpr int WIDE = 16 / (int)sizeof(T);
  const dim3 g(grid), t(THREADS);
  if (interleaved) hipLaunchKernelGGL((qk_norm_kernel<T, WIDE, 1, true, BWD>), g, t, 0, st, a);
  else if (v == WIDE) hipLaunchKernelGGL((qk_norm_kernel<T, WIDE, 1, false, BWD>), g, t, 0, st, a);
  else if (v == 4) hipLaunchKernelGGL((qk_norm_kernel<T, 4, 1, false, BWD>), g, t, 0, st, a);
  else if (v == 2) hipLaunchKernelGGL((qk_norm_kernel<T, 2, 1, false, BWD>), g, t, 0, st, a);
  else hipLaunchKernelGGL((qk_norm_kernel<T, 1, 2, false, BWD>), g, t, 0, st, a);
}

}  // namespace

PPO_EXPORT int ppo_qk_norm_rotary_max_width(void) { return MAX_DIM; }

PPO_EXPORT int ppo_qk_norm_rotary_fwd(void* stream, int dtype, const void* q, const void* k, const int64_t* strides,
                                      const float* q_scale, const float* k_scale, const double* frequencies,
                                      const int32_t* positions, float epsilon, int interleaved, void* q_out,
                                      void* k_out, int batch, int steps, int heads, int kv_heads, int width,
                                      int pairs) {
  const char* what = "ppo_qk_norm_rotary_fwd";
  if (int rc = check(what, dtype, batch, steps, heads, kv_heads, width, pairs)) return rc;
  const int64_t tokens = (int64_t)batch * steps;
  if (tokens == 0 || heads + kv_heads == 0 || width == 0) return PPO_OK;
  if (!strides || (heads > 0 && (!q || !q_out)) || (kv_heads > 0 && (!k || !k_out)) || (pairs > 0 && !frequencies))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  NormArgs a = common_args(epsilon, tokens, steps, width, pairs, interleaved, dtype, heads, kv_heads,
                           frequencies, positions, FWD_ROWS);
  a.part[0] = Rows{q, nullptr, q_scale, q_out, strides[0], strides[1], strides[2], 0, 0, 0, heads, inverse_of(heads)};
  a.part[1] = Rows{k, nullptr, k_scale, k_out, strides[3], strides[4], strides[5], 0, 0, 0, kv_heads,
                   inverse_of(kv_heads)};
  const int v = chunk_columns(dtype, pairs, interleaved);
  const unsigned grid = blocks_of(tokens, a.tile, FWD_BLOCKS);
  if (dtype == NORM_F32) launch_chunk<float, false>(ppo::as_stream(stream), a, v, interleaved != 0, grid);
  else launch_chunk<uint16_t, false>(ppo::as_stream(stream), a, v, interleaved != 0, grid);
  return ppo::check_launch(what);
}

PPO_EXPORT size_t ppo_qk_norm_rotary_bwd_workspace(int width) {
  return width > 0 && width <= MAX_DIM ? sizeof(float) * 2 * (size_t)width * BWD_BLOCKS : 0;
}

PPO_EXPORT int ppo_qk_norm_rotary_bwd(void* stream, int dtype, const void* q, const void* k, const void* dq_out,
                                      const void* dk_out, const int64_t* strides, const float* q_scale,
                                      const float* k_scale, const double* frequencies, const int32_t* positions,
                                      float epsilon, int interleaved, void* dq, void* dk, float* dq_scale,
                                      float* dk_scale, void* workspace, size_t workspace_bytes, int batch, int steps,
                                      int heads, int kv_heads, int width, int pairs) {
  const char* what = "ppo_qk_norm_rotary_bwd";
  if (int rc = check(what, dtype, batch, steps, heads, kv_heads, width, pairs)) return rc;
  if (width == 0) return PPO_OK;
  const int64_t tokens = (int64_t)batch * steps;
  const bool none = tokens == 0 || heads + kv_heads == 0;
  if (!none && (!strides || (heads > 0 && (!q || !dq_out || !dq)) || (kv_heads > 0 && (!k || !dk_out || !dk)) ||
                (pairs > 0 && !frequencies)))
    return ppo::set_error(PPO_ERR_ARG, "%s: null buffer", what);
  const size_t need = ppo_qk_norm_rotary_bwd_workspace(width);
  if (!workspace || workspace_bytes < need)
    return ppo::set_error(PPO_ERR_SPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  int blocks = 0;
  if (!none) {
    NormArgs a = common_args(epsilon, tokens, steps, width, pairs, interleaved, dtype, heads, kv_heads,
                             frequencies, positions, BWD_ROWS);
    a.part[0] = Rows{q, dq_out, q_scale, dq, strides[0], strides[1], strides[2], strides[6], strides[7], strides[8],
                     heads, inverse_of(heads)};
    a.part[1] = Rows{k, dk_out, k_scale, dk, strides[3], strides[4], strides[5], strides[9], strides[10], strides[11],
                     kv_heads, inverse_of(kv_heads)};
    a.partials = static_cast<float*>(workspace);
    const int v = chunk_columns(dtype, pairs, interleaved);
    blocks = (int)blocks_of(tokens, a.tile, BWD_BLOCKS);
    if (dtype == NORM_F32) launch_chunk<float, true>(ppo::as_stream(stream), a, v, interleaved != 0, (unsigned)blocks);
    else launch_chunk<uint16_t, true>(ppo::as_stream(stream), a, v, interleaved != 0, (unsigned)blocks);
  }
  if (dq_scale || dk_scale)
    hipLaunchKernelGGL(qk_norm_scale_kernel, dim3((unsigned)ppo::ceil_div(2 * width, 4)), dim3(256), 0,
                       ppo::as_stream(stream), static_cast<const float*>(workspace), blocks, width, dq_scale, dk_scale);
  return ppo::check_launch(what);
}
