// The end of a transformer block: dropout of the block's output, the
// residual's addition and the root-mean-square norm of the sum, with its
// gradients; or, for serving, the norm's rows in 8 bits with scales.
//
//   h = round(residual + mask x / keep)         the residual stream, stored
//   y = h rstd w,  rstd = 1 / sqrt(mean(h^2) + eps)
//   dh' = dh + rstd (g - n mean(g n)),  g = dy w,  n = h rstd
//   dresidual = dh',  dx = mask dh' / keep,  dw = sum over rows of dy n
//
// The norm is taken of the stored (rounded) h, so the backward needs no other
// copy of it.  The mask is not stored: both directions draw it again from a
// counter-based generator, Philox4x32 with 10 rounds (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): key = the seed,
// counter = (column / 8, row, offset).  Its 128 bits are eight draws of 16
// bits, one per element of a thread's chunk; an element stays where its draw
// reaches drop_least.  16 bits fix the drop probability to a multiple of
// 2^-16, which the factor 65536 / (65536 - drop_least) takes into account.
//
// Bound by the bytes of the rows, each read and written once (and by the latency
// of one row where there are few).  bf16: 131072 rows of 1536 to 8 bits 271 us,
// 5.2 TB/s (a copy of 2 GiB: 4.9); 32768 rows of 1024 with dropout 46 us, 5.8
// TB/s, and backward 64 us, 5.3 TB/s, and 6.5 for dw; 5 rows of 1536 4 us.
#include "common.h"

namespace lsrm {

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t n;
  int hidden;
  float eps;
  uint32_t drop_least;
  float keep_factor;
  const int64_t* rng;   // seed, offset
  int64_t* rng_used;    // their values at the forward
  void *y, *h;
  float* rstd;
  uint8_t* y8;
  float* scales;
  int group_lanes;      // 8-bit rows: lanes (chunks of 8) that share a scale, 0: the row
  // backward
  const void *dy, *dh;
  const float* rstd_in;
  void *dx, *dres, *dw;
  float* dw_part;
};

constexpr int NORM_MAX_HIDDEN = 16384;

// Eight consecutive elements.  Rows of any width and alignment are read and
// written 16 bytes at a time (global accesses need only the alignment of an
// element), a row's last piece element by element.
template <int DT>
struct Chunk {
  typedef uint16_t T;
  struct __attribute__((packed, aligned(2))) V {
    u32x4 w;
  };
  __device__ static inline void ld(const void* p, int64_t i, int cnt, float* v) {
    const T* q = reinterpret_cast<const T*>(p) + i;
    if (cnt >= 8) {
      const u32x4 w = reinterpret_cast<const V*>(q)->w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[2 * k] = to_f32<DT>((uint16_t)(w[k] & 0xffffu));
        v[2 * k + 1] = to_f32<DT>((uint16_t)(w[k] >> 16));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < cnt ? to_f32<DT>(q[k]) : 0.0f;
    }
  }
  __device__ static inline void st(void* p, int64_t i, int cnt, const float* v) {
    T* q = reinterpret_cast<T*>(p) + i;
    if (cnt >= 8) {
      reinterpret_cast<V*>(q)->w = u32x4{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]),
                                         pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < cnt) q[k] = from_f32<DT>(v[k]);
    }
  }
  __device__ static inline float rnd(float v) { return to_f32<DT>(from_f32<DT>(v)); }
};
template <>
struct Chunk<LSRM_F32> {
  struct __attribute__((packed, aligned(4))) V {
    f32x4 w;
  };
  __device__ static inline void ld(const void* p, int64_t i, int cnt, float* v) {
    const float* q = reinterpret_cast<const float*>(p) + i;
    if (cnt >= 8) {
      const f32x4 a = reinterpret_cast<const V*>(q)->w, b = reinterpret_cast<const V*>(q + 4)->w;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = a[k];
        v[4 + k] = b[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < cnt ? q[k] : 0.0f;
    }
  }
  __device__ static inline void st(void* p, int64_t i, int cnt, const float* v) {
    float* q = reinterpret_cast<float*>(p) + i;
    if (cnt >= 8) {
      reinterpret_cast<V*>(q)->w = f32x4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<V*>(q + 4)->w = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < cnt) q[k] = v[k];
    }
  }
  __device__ static inline float rnd(float v) { return v; }
};

__device__ inline void philox(uint32_t col8, uint32_t row, uint64_t seed, uint64_t offset,
                              uint32_t* out) {
  uint32_t c0 = col8, c1 = row, c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0;
  out[1] = c1;
  out[2] = c2;
  out[3] = c3;
}

// v[e] scaled where it stays and 0 where it is dropped.
__device__ inline void drop8(const NormArgs& a, uint32_t col8, uint32_t row, uint64_t seed,
                             uint64_t offset, float* v) {
  uint32_t r[4];
  philox(col8, row, seed, offset, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t d = e % 2 ? r[e / 2] >> 16 : r[e / 2] & 0xffffu;
    v[e] = d >= a.drop_least ? v[e] * a.keep_factor : 0.0f;
  }
}

__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) x += __shfl_xor(x, w);
  return x;
}

// Sum over the W waves of a row (W = 1: the wave's own).
template <int W>
__device__ inline float row_sum(float x, float* s_red) {
  x = wave_sum(x);
  if constexpr (W > 1) {
    __syncthreads();
    if (lane_id() == 0) s_red[wave_id()] = x;
    __syncthreads();
    x = s_red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) x += s_red[i];
  }
  return x;
}

constexpr int NORM_PLAIN = 0, NORM_DROP = 1, NORM_FP8 = 2;

// W = 1: a wave per row, four rows a workgroup; W = 4: a workgroup per row
// (long rows, or few).  A thread holds K chunks of 8 elements, so a row is read
// once and stays in registers.
template <int DT, int K, int W, int MODE>
__global__ __launch_bounds__(256) void residual_norm_kernel(NormArgs a) {
  using C = Chunk<DT>;
  __shared__ float s_red[4];
  const int lane = lane_id(), wv = wave_id();
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wv : blockIdx.x;
  uint64_t seed = 0, offset = 0;
  if constexpr (MODE == NORM_DROP) {
    seed = (uint64_t)a.rng[0];
    offset = (uint64_t)a.rng[1];
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.rng_used[0] = (int64_t)seed;
      a.rng_used[1] = (int64_t)offset;
    }
  }
  if (row >= a.n) return;  // W = 4: the whole workgroup
  const int64_t base = row * a.hidden;
  float h[K][8];
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = ((k * W + (W == 1 ? 0 : wv)) * 64 + lane) * 8, cnt = a.hidden - col;
    if (cnt <= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] = 0.0f;
      continue;
    }
    C::ld(a.x, base + col, cnt, h[k]);
    if constexpr (MODE == NORM_DROP)
      drop8(a, (uint32_t)col / 8, (uint32_t)row, seed, offset, h[k]);
    if (a.residual) {
      float r[8];
      C::ld(a.residual, base + col, cnt, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[k][e] += r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[k][e] = C::rnd(h[k][e]);
      sum = __builtin_fmaf(h[k][e], h[k][e], sum);
    }
    C::st(a.h, base + col, cnt, h[k]);
  }
  const float rstd =
      1.0f / sqrtf(row_sum<W>(sum, s_red) / (float)a.hidden + a.eps);
  if constexpr (MODE != NORM_FP8) {
    if (lane == 0 && (W == 1 || wv == 0)) a.rstd[row] = rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = ((k * W + (W == 1 ? 0 : wv)) * 64 + lane) * 8, cnt = a.hidden - col;
      if (cnt <= 0) continue;
      float w[8];
      C::ld(a.weight, col, cnt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] *= h[k][e] * rstd;
      C::st(a.y, base + col, cnt, w);
    }
  } else {
    // The largest magnitude maps to 448, the largest value of e4m3.
    float top[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = ((k * W + (W == 1 ? 0 : wv)) * 64 + lane) * 8, cnt = a.hidden - col;
      top[k] = 0.0f;
      if (cnt <= 0) continue;
      float w[8];
      C::ld(a.weight, col, cnt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[k][e] = h[k][e] * rstd * w[e];
        top[k] = __builtin_elementwise_maximum(top[k], __builtin_fabsf(h[k][e]));
      }
    }
    if (a.group_lanes == 0) {
      float m = top[0];
#pragma unroll
      for (int k = 1; k < K; ++k) m = __builtin_elementwise_maximum(m, top[k]);
      for (int w = 32; w > 0; w >>= 1)
        m = __builtin_elementwise_maximum(m, __shfl_xor(m, w));
      if constexpr (W > 1) {
        __syncthreads();
        if (lane == 0) s_red[wv] = m;
        __syncthreads();
        m = s_red[0];
#pragma unroll
        for (int i = 1; i < W; ++i) m = __builtin_elementwise_maximum(m, s_red[i]);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) top[k] = m;
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
        for (int w = a.group_lanes >> 1; w > 0; w >>= 1)
          top[k] = __builtin_elementwise_maximum(top[k], __shfl_xor(top[k], w));
    }
    const int groups = a.group_lanes ? a.hidden / (8 * a.group_lanes) : 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int chunk = (k * W + (W == 1 ? 0 : wv)) * 64 + lane, col = chunk * 8;
      const int cnt = a.hidden - col;
      if (cnt <= 0) continue;
      const float scale = top[k] == 0.0f ? 1.0f : top[k] / 448.0f, inv = 1.0f / scale;
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] = h[k][e] * inv;  // a NaN stays one
        q[e] = q[e] > 448.0f ? 448.0f : (q[e] < -448.0f ? -448.0f : q[e]);
      }
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
      int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
      uint8_t* out = a.y8 + base + col;
      if (cnt >= 8) {
        struct __attribute__((packed, aligned(1))) V {
          u32x2 w;
        };
        reinterpret_cast<V*>(out)->w = u32x2{(uint32_t)lo, (uint32_t)hi};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < cnt) out[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
      }
      if (a.group_lanes == 0) {
        if (chunk == 0) a.scales[row] = scale;
      } else if (chunk % a.group_lanes == 0) {
        a.scales[row * groups + chunk / a.group_lanes] = scale;
      }
    }
  }
}

// Rows blockIdx.x * (4 / W) + .., stepping by the grid; dw_part[blockIdx.x]
// receives the workgroup's sum of dy n, its waves' rows in a fixed order.
template <int DT, int K, int W, bool DROP>
__global__ __launch_bounds__(256) void residual_norm_bwd_kernel(NormArgs a) {
  using C = Chunk<DT>;
  __shared__ float s_red[4];
  extern __shared__ float s_dw[];  // W = 1: [4][hidden rounded up to 8]
  const int lane = lane_id(), wv = wave_id();
  uint64_t seed = 0, offset = 0;
  if constexpr (DROP) {
    seed = (uint64_t)a.rng[0];
    offset = (uint64_t)a.rng[1];
  }
  float dw[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[k][e] = 0.0f;
  constexpr int RPB = 4 / W;
  for (int64_t row = (int64_t)blockIdx.x * RPB + (W == 1 ? wv : 0); row < a.n;
       row += (int64_t)gridDim.x * RPB) {
    const int64_t base = row * a.hidden;
    const float rstd = a.rstd_in[row];
    float n[K][8], g[K][8];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = ((k * W + (W == 1 ? 0 : wv)) * 64 + lane) * 8, cnt = a.hidden - col;
      if (cnt <= 0 || !a.dy) {
#pragma unroll
        for (int e = 0; e < 8; ++e) n[k][e] = g[k][e] = 0.0f;
        continue;
      }
      float w[8];
      C::ld(a.h, base + col, cnt, n[k]);
      C::ld(a.dy, base + col, cnt, g[k]);
      C::ld(a.weight, col, cnt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[k][e] *= rstd;
        dw[k][e] = __builtin_fmaf(g[k][e], n[k][e], dw[k][e]);
        g[k][e] *= w[e];
        sum = __builtin_fmaf(g[k][e], n[k][e], sum);
      }
    }
    const float mean = row_sum<W>(sum, s_red) / (float)a.hidden;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = ((k * W + (W == 1 ? 0 : wv)) * 64 + lane) * 8, cnt = a.hidden - col;
      if (cnt <= 0) continue;
      float d[8];
      if (a.dh) {
        C::ld(a.dh, base + col, cnt, d);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        d[e] = __builtin_fmaf(rstd, g[k][e] - n[k][e] * mean, d[e]);
      C::st(a.dres, base + col, cnt, d);
      if constexpr (DROP) {
        drop8(a, (uint32_t)col / 8, (uint32_t)row, seed, offset, d);
        C::st(a.dx, base + col, cnt, d);
      }
    }
  }
  float* part = a.dw_part + (int64_t)blockIdx.x * a.hidden;
  if constexpr (W == 1) {
    const int stride = (a.hidden + 7) / 8 * 8;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * 64 + lane) * 8;
      if (col < a.hidden)
#pragma unroll
        for (int e = 0; e < 8; ++e) s_dw[wv * stride + col + e] = dw[k][e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.hidden; c += 256)
      part[c] = s_dw[c] + s_dw[stride + c] + s_dw[2 * stride + c] + s_dw[3 * stride + c];
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = ((k * W + wv) * 64 + lane) * 8, cnt = a.hidden - col;
      if (cnt > 0) Chunk<LSRM_F32>::st(part, col, cnt, dw[k]);
    }
  }
}

// dw: 16 columns a workgroup (64 bytes of a partial sum); 64 threads a column
// take every 64th partial sum, then their sums in order.
template <int DT>
__global__ __launch_bounds__(1024) void residual_norm_dw_kernel(NormArgs a, int parts) {
  __shared__ float s[64][17];
  const int col = threadIdx.x & 15, at = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + col;
  float sum = 0.0f;
  if (c < a.hidden)
    for (int p = at; p < parts; p += 64) sum += a.dw_part[(int64_t)p * a.hidden + c];
  s[at][col] = sum;
  __syncthreads();
  if (at == 0 && c < a.hidden) {
    for (int w = 1; w < 64; ++w) sum += s[w][col];
    if constexpr (DT == LSRM_F32)
      reinterpret_cast<float*>(a.dw)[c] = sum;
    else
      reinterpret_cast<uint16_t*>(a.dw)[c] = from_f32<DT>(sum);
  }
}

// A wave or a workgroup for a row.  Long rows leave a wave few rows in flight,
// and few rows leave the card empty.  bf16 forward, a wave against a workgroup:
// 16384 rows of 512 10.5 us against 18.3, of 1536 24.3 against 25.4, of 4096 87
// against 77; 1024 rows of 512 3.2 against 3.5, of 1536 4.9 against 4.1, of 2048
// 5.9 against 4.5.  The backward holds three times as much of a row: 16384 rows
// of 512 21 against 37, of 1536 51 against 45, of 2048 64 against 49; 256 rows of
// 512 5.9 against 7.0, of 2048 10.5 against 8.4.
static int norm_waves(int64_t n, int64_t hidden) { return hidden > 2048 || n < hidden ? 4 : 1; }
static int norm_bwd_waves(int64_t n, int64_t hidden) { return hidden > 1024 || n < 1024 ? 4 : 1; }
static int norm_chunks(int64_t hidden, int waves) {
  const int64_t k = (hidden + 512 * waves - 1) / (512 * waves);
  return k <= 2 ? 2 : (k <= 4 ? 4 : 8);
}

// Workgroups of the backward, each with one partial sum of dw, written and read
// again: two to four per CU, the larger number where each has two turns at least
// (1024 rows of 2048: 512 workgroups 13.5 us, 1024 17.8; 16384 rows of 2048: 64
// and 49).
static int norm_bwd_groups(int64_t n, int64_t hidden) {
  const int64_t need = norm_bwd_waves(n, hidden) == 1 ? (n + 3) / 4 : n;
  if (need <= 512) return (int)(need > 0 ? need : 1);
  return (int)(need / 2 < 512 ? 512 : (need / 2 < 1024 ? need / 2 : 1024));
}

template <int DT, int MODE>
static int norm_launch(const NormArgs& a, hipStream_t st) {
  const int w = norm_waves(a.n, a.hidden), k = norm_chunks(a.hidden, w);
  const dim3 grid((unsigned)(w == 1 ? (a.n + 3) / 4 : a.n)), block(256);
#define LSRM_NORM(KV, WV) \
  hipLaunchKernelGGL((residual_norm_kernel<DT, KV, WV, MODE>), grid, block, 0, st, a)
  if (w == 1) {
    if (k == 2) LSRM_NORM(2, 1);
    else LSRM_NORM(4, 1);
  } else {
    if (k == 2) LSRM_NORM(2, 4);
    else if (k == 4) LSRM_NORM(4, 4);
    else LSRM_NORM(8, 4);
  }
#undef LSRM_NORM
  LSRM_CHECK_LAUNCH();
  return LSRM_OK;
}

template <int DT, bool DROP>
static int norm_bwd_launch(const NormArgs& a, hipStream_t st) {
  const int w = norm_bwd_waves(a.n, a.hidden), k = norm_chunks(a.hidden, w);
  const int groups = norm_bwd_groups(a.n, a.hidden);
  const size_t lds = w == 1 ? (size_t)(a.hidden + 7) / 8 * 8 * 16 : 0;
  const dim3 grid(groups), block(256);
#define LSRM_NORM(KV, WV) \
  hipLaunchKernelGGL((residual_norm_bwd_kernel<DT, KV, WV, DROP>), grid, block, lds, st, a)
  if (w == 1) {
    LSRM_NORM(2, 1);
  } else {
    if (k == 2) LSRM_NORM(2, 4);
    else if (k == 4) LSRM_NORM(4, 4);
    else LSRM_NORM(8, 4);
  }
#undef LSRM_NORM
  LSRM_CHECK_LAUNCH();
  hipLaunchKernelGGL(residual_norm_dw_kernel<DT>, dim3((a.hidden + 15) / 16), dim3(1024), 0, st,
                     a, groups);
  LSRM_CHECK_LAUNCH();
  return LSRM_OK;
}

static int norm_check(int dtype, int64_t n, int64_t hidden, const void* const* ptrs, int count) {
  if (dtype != LSRM_BF16 && dtype != LSRM_F16 && dtype != LSRM_F32) return LSRM_ERR_UNSUPPORTED;
  if (n < 0 || hidden <= 0) return LSRM_ERR_INVALID_ARG;
  if (hidden > NORM_MAX_HIDDEN || n > (int64_t{1} << 30)) return LSRM_ERR_UNSUPPORTED;
  const uintptr_t align = dtype == LSRM_F32 ? 3u : 1u;
  for (int i = 0; i < count; ++i) {
    if (n > 0 && !ptrs[i]) return LSRM_ERR_INVALID_ARG;
    if ((uintptr_t)ptrs[i] & align) return LSRM_ERR_INVALID_ARG;
  }
  return LSRM_OK;
}

}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_residual_norm_fwd(const void* x, const void* residual, const void* weight,
                                      int dtype, int64_t n_tokens, int64_t hidden, float eps,
                                      int drop_least, const int64_t* rng, int64_t* rng_used,
                                      void* y, void* h, float* rstd, void* stream) {
  const void* ptrs[4] = {x, weight, y, h};
  const int rc = norm_check(dtype, n_tokens, hidden, ptrs, 4);
  if (rc) return rc;
  if (drop_least < 0 || drop_least > 65535 || !(eps >= 0.0f) ||
      (drop_least > 0 && (!rng || !rng_used)) || (n_tokens > 0 && !rstd))
    return LSRM_ERR_INVALID_ARG;
  if (n_tokens == 0) return LSRM_OK;
  NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.n = n_tokens;
  a.hidden = (int)hidden;
  a.eps = eps;
  a.drop_least = (uint32_t)drop_least;
  a.keep_factor = 65536.0f / (float)(65536 - drop_least);
  a.rng = rng;
  a.rng_used = rng_used;
  a.y = y;
  a.h = h;
  a.rstd = rstd;
  hipStream_t st = (hipStream_t)stream;
#define LSRM_NORM_DT(DT)                                         \
  return drop_least > 0 ? norm_launch<DT, NORM_DROP>(a, st) : \
                          norm_launch<DT, NORM_PLAIN>(a, st)
  if (dtype == LSRM_BF16) LSRM_NORM_DT(LSRM_BF16);
  if (dtype == LSRM_F16) LSRM_NORM_DT(LSRM_F16);
  LSRM_NORM_DT(LSRM_F32);
#undef LSRM_NORM_DT
}

extern "C" int lsrm_residual_norm_fp8(const void* x, const void* residual, const void* weight,
                                      int dtype, int64_t n_tokens, int64_t hidden, float eps,
                                      int64_t group, void* y8, float* scales, void* h,
                                      void* stream) {
  const void* ptrs[3] = {x, weight, h};
  const int rc = norm_check(dtype, n_tokens, hidden, ptrs, 3);
  if (rc) return rc;
  if (!(eps >= 0.0f) || (n_tokens > 0 && (!y8 || !scales)) ||
      (group != 0 && (group < 0 || hidden % group != 0)))
    return LSRM_ERR_INVALID_ARG;
  if (group != 0 && group != 32 && group != 64 && group != 128) return LSRM_ERR_UNSUPPORTED;
  if (n_tokens == 0) return LSRM_OK;
  NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.n = n_tokens;
  a.hidden = (int)hidden;
  a.eps = eps;
  a.h = h;
  a.y8 = (uint8_t*)y8;
  a.scales = scales;
  a.group_lanes = (int)(group / 8);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSRM_BF16) return norm_launch<LSRM_BF16, NORM_FP8>(a, st);
  if (dtype == LSRM_F16) return norm_launch<LSRM_F16, NORM_FP8>(a, st);
  return norm_launch<LSRM_F32, NORM_FP8>(a, st);
}

extern "C" size_t lsrm_residual_norm_bwd_workspace_size(int64_t n_tokens, int64_t hidden) {
  if (n_tokens < 0 || hidden <= 0 || hidden > NORM_MAX_HIDDEN) return 0;
  return (size_t)norm_bwd_groups(n_tokens, hidden) * hidden * sizeof(float) + 256;
}

extern "C" int lsrm_residual_norm_bwd(const void* dy, const void* dh, const void* h,
                                      const void* weight, const float* rstd, int dtype,
                                      int64_t n_tokens, int64_t hidden, int drop_least,
                                      const int64_t* rng, void* dx, void* d_residual,
                                      void* d_weight, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const void* ptrs[3] = {h, weight, d_residual};
  const int rc = norm_check(dtype, n_tokens, hidden, ptrs, 3);
  if (rc) return rc;
  const uintptr_t align = dtype == LSRM_F32 ? 3u : 1u;
  if (drop_least < 0 || drop_least > 65535 || (drop_least > 0) != (dx != nullptr) ||
      (drop_least > 0 && !rng) || !d_weight || (n_tokens > 0 && !rstd) ||
      (((uintptr_t)dy | (uintptr_t)dh | (uintptr_t)dx | (uintptr_t)d_weight) & align))
    return LSRM_ERR_INVALID_ARG;
  Carver c{(char*)workspace, 0, workspace_bytes};
  NormArgs a{};
  a.dw_part = c.take<float>((size_t)norm_bwd_groups(n_tokens, hidden) * hidden);
  if (!workspace || !c.ok()) return LSRM_ERR_WORKSPACE;
  a.weight = weight;
  a.n = n_tokens;
  a.hidden = (int)hidden;
  a.drop_least = (uint32_t)drop_least;
  a.keep_factor = 65536.0f / (float)(65536 - drop_least);
  a.rng = rng;
  a.h = const_cast<void*>(h);
  a.dy = dy;
  a.dh = dh;
  a.rstd_in = rstd;
  a.dx = dx;
  a.dres = d_residual;
  a.dw = d_weight;
  hipStream_t st = (hipStream_t)stream;
#define LSRM_NORM_DT(DT) \
  return drop_least > 0 ? norm_bwd_launch<DT, true>(a, st) : norm_bwd_launch<DT, false>(a, st)
  if (dtype == LSRM_BF16) LSRM_NORM_DT(LSRM_BF16);
  if (dtype == LSRM_F16) LSRM_NORM_DT(LSRM_F16);
  LSRM_NORM_DT(LSRM_F32);
#undef LSRM_NORM_DT
}
