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
// A workgroup takes a tile of steps with all heads of both: the angles' sines and cosines
// are formed once a step and pair (p f in float64, since float32 is off by up
// to p 2^-24 radians, and its turns brought below one before the float32
// sine) and read from LDS by every head.  L lanes hold a row, each in units of
// two chunks of VW columns that hold whole pairs, so the rotation needs no
// lane exchange; the sums over a row are L-lane butterflies in float32.
// Bound by HBM: x is read and out written once.
#include "split_f32.h"

#include <algorithm>

namespace {

enum NormDtype { NORM_F32 = 0, NORM_BF16 = 1 };

constexpr int THREADS = 256;
constexpr int MAX_DIM = 256, MAX_PAIRS = MAX_DIM / 2;
constexpr int MAX_TILE = 16;    // steps of a tile
constexpr int BWD_BLOCKS = 1024;  // most workgroups of the backward launch, each with its partial sums of dscale

struct Rows {
  const void* x;
  const void* cot;      // backward
  const float* scale;   // [D], or null (ones)
  void* out;            // [tokens, heads, D]
  int64_t sb, st, sh;   // element strides of x
  int64_t cb, ct, ch;   // and of cot
  int heads;
};

struct NormArgs {
  Rows part[2];         // queries, keys
  const double* frequencies;
  const int32_t* positions;  // [batch, steps], or null (the step itself)
  float* partials;      // backward: [workgroups, 2, D]
  float eps;
  uint32_t tokens, steps;
  int D, P, interleaved, tile, lanes_log2;
};

__device__ __forceinline__ float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
__device__ __forceinline__ float widen(float x) { return x; }

template <int VW> __device__ __forceinline__ void load_row(const uint16_t* p, int left, float (&v)[VW]) {
  uint16_t e[VW];
  if (left >= VW) {
    __builtin_memcpy(e, p, 2 * VW);
  } else {
#pragma unroll
    for (int j = 0; j < VW; ++j) e[j] = j < left ? p[j] : (uint16_t)0;
  }
#pragma unroll
  for (int j = 0; j < VW; ++j) v[j] = widen(e[j]);
}
template <int VW> __device__ __forceinline__ void load_row(const float* p, int left, float (&v)[VW]) {
  if (left >= VW) {
    __builtin_memcpy(v, p, 4 * VW);
  } else {
#pragma unroll
    for (int j = 0; j < VW; ++j) v[j] = j < left ? p[j] : 0.f;
  }
}
template <int VW> __device__ __forceinline__ void store_row(uint16_t* p, int left, const float (&v)[VW]) {
  uint16_t e[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) e[j] = (uint16_t)ppo::pack_bf16(v[j], v[j]);
  if constexpr (VW >= 2) {
    if (left >= VW) {
      uint32_t w[VW / 2];
#pragma unroll
      for (int j = 0; j < VW / 2; ++j) w[j] = ppo::pack_bf16(v[2 * j], v[2 * j + 1]);
      __builtin_memcpy(p, w, 2 * VW);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < VW; ++j)
    if (j < left) p[j] = e[j];
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

// The columns of a lane's unit u: chunks at a and b.  Columns of pairs come
// first; in the layout of halves a chunk of first columns and that of their
// partners, otherwise two neighbouring chunks.
struct Unit {
  int a, b, pair;  // pair: the first pair of the unit's first chunk, or -1 (no rotation)
};
template <int VW> __device__ __forceinline__ Unit unit_of(int u, int P, int interleaved) {
  Unit r;
  if (interleaved) {
    r.a = 2 * VW * u;
    r.b = r.a + VW;
    r.pair = r.a < 2 * P ? VW * u : -1;
  } else if (u * VW < P) {
    r.a = u * VW;
    r.b = P + r.a;
    r.pair = r.a;
  } else {
    r.a = 2 * VW * u;  // past the pairs' 2 VW (P / VW) columns
    r.b = r.a + VW;
    r.pair = -1;
  }
  return r;
}

// (a, b) turned by the unit's angles, back for `sign` -1.
template <int VW>
__device__ __forceinline__ void turn(float (&a)[VW], float (&b)[VW], const Unit& u, const float2* cs, int P,
                                     int interleaved, float sign) {
  if (u.pair < 0) return;
  if (interleaved) {
    if constexpr (VW >= 2) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float(&v)[VW] = c ? b : a;
#pragma unroll
        for (int j = 0; j < VW / 2; ++j) {
          const int i = u.pair + c * (VW / 2) + j;
          if (i < P) {
            const float2 w = cs[i];
            const float s = sign * w.y, x = v[2 * j], y = v[2 * j + 1];
            v[2 * j] = x * w.x - y * s;
            v[2 * j + 1] = y * w.x + x * s;
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      const float2 w = cs[u.pair + j];
      const float s = sign * w.y, x = a[j], y = b[j];
      a[j] = x * w.x - y * s;
      b[j] = y * w.x + x * s;
    }
  }
}

template <typename T, int VW, int UPL, bool BWD>
__global__ void __launch_bounds__(THREADS) qk_norm_kernel(NormArgs p) {
  __shared__ float2 cs[MAX_TILE * MAX_PAIRS];
  __shared__ int64_t at[4][MAX_TILE];   // element offsets of a step's rows: x of both parts, cotangents of both
  __shared__ float red[BWD ? 2 * VW * UPL * THREADS : 1];
  const int tid = threadIdx.x, L = 1 << p.lanes_log2, l = tid & (L - 1), D = p.D, P = p.P;
  Unit unit[UPL];
#pragma unroll
  for (int k = 0; k < UPL; ++k) unit[k] = unit_of<VW>(l + k * L, P, p.interleaved);
  float sum[2][UPL][2][VW];
  if constexpr (BWD) {
#pragma unroll
    for (int i = 0; i < 2 * UPL * 2 * VW; ++i) (&sum[0][0][0][0])[i] = 0.f;
  }
  const uint32_t tiles = (p.tokens + p.tile - 1) / p.tile;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint32_t t0 = tile * p.tile;
    const int n = (int)min((uint32_t)p.tile, p.tokens - t0);
    for (int i = tid; i < n * P; i += THREADS) {
      const int s = i / P, f = i - s * P;
      const uint32_t token = t0 + s;
      const double pos = p.positions ? (double)p.positions[token] : (double)(token % p.steps);
      double turns = pos * p.frequencies[f] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      float sn, cn;
      sincospif(2.f * (float)turns, &sn, &cn);
      cs[s * P + f] = make_float2(cn, sn);
    }
    if (tid < n) {
      const uint32_t token = t0 + tid, b = token / p.steps, t = token - b * p.steps;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        at[w][tid] = (int64_t)b * p.part[w].sb + (int64_t)t * p.part[w].st;
        if constexpr (BWD) at[2 + w][tid] = (int64_t)b * p.part[w].cb + (int64_t)t * p.part[w].ct;
      }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Rows& q = p.part[w];
      float wa[UPL][VW], wb[UPL][VW];
#pragma unroll
      for (int k = 0; k < UPL; ++k)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          wa[k][j] = q.scale && unit[k].a + j < D ? q.scale[unit[k].a + j] : 1.f;
          wb[k][j] = q.scale && unit[k].b + j < D ? q.scale[unit[k].b + j] : 1.f;
        }
      const int rows = n * q.heads;
      for (int r = tid >> p.lanes_log2; r < rows; r += THREADS >> p.lanes_log2) {
        const int s = r / q.heads, h = r - s * q.heads;
        const T* x = static_cast<const T*>(q.x) + at[w][s] + h * q.sh;
        T* out = static_cast<T*>(q.out) + ((int64_t)(t0 + s) * q.heads + h) * D;
        float a[UPL][VW], b[UPL][VW];
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
          load_row<VW>(x + unit[k].a, D - unit[k].a, a[k]);
          load_row<VW>(x + unit[k].b, D - unit[k].b, b[k]);
        }
        float ca[UPL][VW], cb[UPL][VW];
        if constexpr (BWD) {
          const T* c = static_cast<const T*>(q.cot) + at[2 + w][s] + h * q.ch;
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            load_row<VW>(c + unit[k].a, D - unit[k].a, ca[k]);
            load_row<VW>(c + unit[k].b, D - unit[k].b, cb[k]);
          }
        }
#pragma unroll
        for (int k = 0; k < UPL; ++k)
#pragma unroll
          for (int j = 0; j < VW; ++j) ss = __fmaf_rn(a[k][j], a[k][j], __fmaf_rn(b[k][j], b[k][j], ss));
        ss = lanes_sum(ss, p.lanes_log2);
        const float rstd = 1.f / sqrtf(ss / (float)D + p.eps);
        if constexpr (!BWD) {
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
#pragma unroll
            for (int j = 0; j < VW; ++j) {
              a[k][j] = a[k][j] * rstd * wa[k][j];
              b[k][j] = b[k][j] * rstd * wb[k][j];
            }
            turn<VW>(a[k], b[k], unit[k], cs + s * P, P, p.interleaved, 1.f);
            store_row<VW>(out + unit[k].a, D - unit[k].a, a[k]);
            store_row<VW>(out + unit[k].b, D - unit[k].b, b[k]);
          }
        } else {
          float m = 0.f;
#pragma unroll
          for (int k = 0; k < UPL; ++k) {
            turn<VW>(ca[k], cb[k], unit[k], cs + s * P, P, p.interleaved, -1.f);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
              a[k][j] *= rstd;
              b[k][j] *= rstd;
              sum[w][k][0][j] = __fmaf_rn(ca[k][j], a[k][j], sum[w][k][0][j]);
              sum[w][k][1][j] = __fmaf_rn(cb[k][j], b[k][j], sum[w][k][1][j]);
              ca[k][j] *= wa[k][j];
              cb[k][j] *= wb[k][j];
              m = __fmaf_rn(ca[k][j], a[k][j], __fmaf_rn(cb[k][j], b[k][j], m));
            }
          }
          m = lanes_sum(m, p.lanes_log2) / (float)D;
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
    }
    __syncthreads();
  }
  if constexpr (BWD) {
    // this workgroup's sums of dscale: a row group's lanes side by side, added
    // in the groups' order
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      constexpr int PER = 2 * VW * UPL;
#pragma unroll
      for (int k = 0; k < UPL; ++k)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          red[(k * 2 * VW + j) * THREADS + tid] = sum[w][k][0][j];
          red[(k * 2 * VW + VW + j) * THREADS + tid] = sum[w][k][1][j];
        }
      __syncthreads();
      for (int i = tid; i < PER * L; i += THREADS) {
        const int e = i >> p.lanes_log2, ll = i & (L - 1);
        float s = 0.f;
        for (int g = ll; g < THREADS; g += L) s += red[e * THREADS + g];
        const int k = e / (2 * VW), j = e % (2 * VW);
        const Unit u = unit_of<VW>(ll + k * L, P, p.interleaved);
        const int col = j < VW ? u.a + j : u.b + j - VW;
        if (col < D) p.partials[((int64_t)blockIdx.x * 2 + w) * D + col] = s;
      }
      __syncthreads();
    }
  }
}

// dscale of both parts: the workgroups' sums, 16 columns by 16 groups of them
// a workgroup, added in a fixed order.
__global__ void __launch_bounds__(256) qk_norm_scale_kernel(const float* partials, int blocks, int D, float* dq_scale,
                                                            float* dk_scale) {
  __shared__ float part[16][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < 2 * D)
    for (int b = g; b < blocks; b += 16) s += partials[(int64_t)b * 2 * D + col];
  part[g][c] = s;
  __syncthreads();
  if (g == 0 && col < 2 * D) {
    s = 0.f;
    for (int i = 0; i < 16; ++i) s += part[i][c];
    float* out = col < D ? dq_scale : dk_scale;
    if (out) out[col < D ? col : col - D] = s;
  }
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

int lanes_log2_of(int D, int v) {
  int log2 = 0;
  while (log2 < 6 && (2 * v << log2) < D) ++log2;
  return log2;
}

// Steps of a tile: enough rows to keep the workgroup busy, but a tile for
// every compute unit where there are few.
int tile_of(int64_t tokens, int rows, int lanes_log2) {
  const int64_t busy = std::max<int64_t>(1, 2048 / ((int64_t)rows << lanes_log2));
  return (int)std::max<int64_t>(1, std::min<int64_t>({busy, MAX_TILE, ppo::ceil_div64(tokens, 512)}));
}

int blocks_of(int64_t tokens, int tile) {
  return (int)std::min<int64_t>(BWD_BLOCKS, std::max<int64_t>(1, ppo::ceil_div64(tokens, tile)));
}

int check(const char* what, int dtype, int batch, int steps, int heads, int kv_heads, int dim, int pairs) {
  if (dtype != NORM_F32 && dtype != NORM_BF16) return ppo::set_error(PPO_ERR_ARG, "%s: bad dtype %d", what, dtype);
  if (batch < 0 || steps < 0 || heads < 0 || kv_heads < 0 || dim < 0 || pairs < 0 || 2 * (int64_t)pairs > dim)
    return ppo::set_error(PPO_ERR_ARG, "%s: bad size (batch %d steps %d heads %d, %d width %d pairs %d)", what, batch,
                          steps, heads, kv_heads, dim, pairs);
  if (dim > MAX_DIM) return ppo::set_error(PPO_ERR_ARG, "%s: width %d above %d", what, dim, MAX_DIM);
  if ((int64_t)heads + kv_heads > 65536) return ppo::set_error(PPO_ERR_ARG, "%s: more than 65536 heads", what);
  if ((int64_t)batch * steps > INT32_MAX) return ppo::set_error(PPO_ERR_ARG, "%s: batch x steps above 2^31 - 1", what);
  return PPO_OK;
}

template <typename T, bool BWD>
void launch_chunk(hipStream_t st, const NormArgs& a, int v, unsigned grid) {
  const dim3 g(grid), t(THREADS);
  if constexpr (sizeof(T) == 2) {
    if (v == 8) {
      hipLaunchKernelGGL((qk_norm_kernel<T, 8, 1, BWD>), g, t, 0, st, a);
      return;
    }
  }
  if (v == 4) hipLaunchKernelGGL((qk_norm_kernel<T, 4, 1, BWD>), g, t, 0, st, a);
  else if (v == 2) hipLaunchKernelGGL((qk_norm_kernel<T, 2, 1, BWD>), g, t, 0, st, a);
  else hipLaunchKernelGGL((qk_norm_kernel<T, 1, 2, BWD>), g, t, 0, st, a);
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
  NormArgs a{};
  a.part[0] = Rows{q, nullptr, q_scale, q_out, strides[0], strides[1], strides[2], 0, 0, 0, heads};
  a.part[1] = Rows{k, nullptr, k_scale, k_out, strides[3], strides[4], strides[5], 0, 0, 0, kv_heads};
  a.frequencies = frequencies;
  a.positions = positions;
  a.eps = epsilon;
  a.tokens = (uint32_t)tokens;
  a.steps = (uint32_t)steps;
  a.D = width;
  a.P = pairs;
  a.interleaved = interleaved != 0;
  const int v = chunk_columns(dtype, pairs, a.interleaved);
  a.lanes_log2 = lanes_log2_of(width, v);
  a.tile = tile_of(tokens, heads + kv_heads, a.lanes_log2);
  const unsigned grid = (unsigned)ppo::ceil_div64(tokens, a.tile);
  if (dtype == NORM_F32) launch_chunk<float, false>(ppo::as_stream(stream), a, v, grid);
  else launch_chunk<uint16_t, false>(ppo::as_stream(stream), a, v, grid);
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
    NormArgs a{};
    a.part[0] = Rows{q, dq_out, q_scale, dq, strides[0], strides[1], strides[2], strides[6], strides[7], strides[8],
                     heads};
    a.part[1] = Rows{k, dk_out, k_scale, dk, strides[3], strides[4], strides[5], strides[9], strides[10], strides[11],
                     kv_heads};
    a.frequencies = frequencies;
    a.positions = positions;
    a.partials = static_cast<float*>(workspace);
    a.eps = epsilon;
    a.tokens = (uint32_t)tokens;
    a.steps = (uint32_t)steps;
    a.D = width;
    a.P = pairs;
    a.interleaved = interleaved != 0;
    const int v = chunk_columns(dtype, pairs, a.interleaved);
    a.lanes_log2 = lanes_log2_of(width, v);
    a.tile = tile_of(tokens, heads + kv_heads, a.lanes_log2);
    blocks = blocks_of(tokens, a.tile);
    if (dtype == NORM_F32) launch_chunk<float, true>(ppo::as_stream(stream), a, v, (unsigned)blocks);
    else launch_chunk<uint16_t, true>(ppo::as_stream(stream), a, v, (unsigned)blocks);
  }
  if (dq_scale || dk_scale)
    hipLaunchKernelGGL(qk_norm_scale_kernel, dim3((unsigned)ppo::ceil_div(2 * width, 16)), dim3(256), 0,
                       ppo::as_stream(stream), static_cast<const float*>(workspace), blocks, width, dq_scale, dk_scale);
  return ppo::check_launch(what);
}
