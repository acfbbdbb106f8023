// Sliding-window attention backward on bf16/fp16 MFMA (gfx950).
//
//   P = exp2(scale log2(e) Q K^T + bias - LSE),  dV = P^T dO,
//   dP = dO V^T,  dS = P (dP - rowsum(dO O)),
//   dQ = scale dS K,  dK = scale dS^T Q,
//   dtable[b, head] = the sum of dS over the positions of bucket b.
//
// Two kernels recompute P: one per query tile (dQ, and the sums of dS per
// relative position), one per key tile (dK and dV); every output has one
// writer and every sum a fixed order.
#include "window.h"

namespace lsrm {

int win_args(WinArgs& a, const void* q, const void* k, const void* v, int dtype, int64_t q_stride,
             int64_t k_stride, int64_t v_stride, int64_t nq, int64_t nk, int64_t hq, int64_t hkv,
             int64_t d, const int32_t* cu_q, const int32_t* cu_k, int64_t batch, int64_t left,
             int64_t right, int64_t sinks, const void* table, int64_t n_buckets,
             const int32_t* buckets, int64_t range, float scale);

// Sums of a 32 x 32 block of dS along its diagonals (one relative position
// each) go through LDS: element (key j, query i) is stored at row j + 31 - i,
// column i, and lane r adds up row r.  A row's unused places stay 0.  Rows of
// 36 words put 16 lanes' 16-byte reads, and 32 lanes' writes 35 words apart, on
// different banks.  (Adding the elements to the sums with LDS float atomics,
// one half of the wave at a time, took 85 cycles an instruction: the kernel
// 979 us at 32768 tokens, 16 heads, 511 keys, R = 128; this way %SKEW_US% us.)
constexpr int SKEW_ROWS = 63, SKEW_PITCH = 36, SKEW_WORDS = SKEW_ROWS * SKEW_PITCH + 4;

template <int DT, int D, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 4))) void
window_dq_kernel(WinArgs a) {
  using G = KvTile<D>;
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ __align__(1024) char sK[2][G::BYTES];
  __shared__ __align__(1024) char sV[2][G::BYTES];
  extern __shared__ float s_dyn[];  // BIAS: bias of the heads, then sums of the waves

  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
  const int hb = lane >> 5, l32 = lane & 31;
  const int item = win_item();
  const int groups = a.g >> a.gt_log2;
  if (item >= a.n_tiles * a.hkv * groups) return;
  const int head_group = item / a.n_tiles, tile = item % a.n_tiles;
  const int h = head_group / groups;
  const int gt = 1 << a.gt_log2, gt_mask = gt - 1;
  const int head0 = h * a.g + (head_group % groups) * gt, hh = head0 + (wv & gt_mask);
  const int tq = 128 >> a.gt_log2;
  const int len = BIAS ? win_bias_len(a.range) : 0, n_pos = 2 * a.range + 1;
  float* s_bins = s_dyn + gt * len;
  float* s_skew = s_bins + 4 * len + (-(gt * len + 4 * len) & 3);  // 16-byte aligned
  int idx;
  WinSeq s = win_sequence(a, win_find(a.cu_q, a.batch, a.nq, tq, tile, &idx));
  if (s.b >= a.batch) s.lk = 0;
  if (idx < 0 || (int64_t)idx * tq >= s.lq) {
    if constexpr (BIAS) {  // every tile's sums are read
      for (int i = tid; i < gt * n_pos; i += 256)
        a.bias_part[((int64_t)tile * a.hq + head0) * n_pos + i] = 0.0f;
    }
    return;
  }
  const int i0 = idx * tq, lk = s.lk;
  const int qn = s.lq - i0 < tq ? s.lq - i0 : tq;
  const int r0 = (wv >> a.gt_log2) * 32;
  const bool row_ok = r0 + l32 < qn;
  const int pos0 = i0 + lk - s.lq;
  const int64_t qi = (int64_t)s.q0 + i0 + r0 + l32;
  const int p_last = pos0 + qn - 1;
  const int lo = pos0 - a.left > 0 ? pos0 - a.left : 0;
  int hi = p_last + a.right + 1;
  hi = hi < lk ? hi : lk;
  const int ns = hi > 0 ? (a.sinks < lo ? a.sinks : lo) : 0;
  const int st = ns > 0 ? 1 : 0;
  const int nt = st + (hi > lo ? (hi - lo + KT - 1) / KT : 0);
  const int w_first = pos0 + r0, w_last = w_first + 31 < p_last ? w_first + 31 : p_last;
  const bool wave_on = r0 < qn;
  const int w_lo = w_first - a.left;
  int w_hi = w_last + a.right + 1;
  w_hi = w_hi < lk ? w_hi : lk;
  const int p = w_first + l32;
  const int row_lo = p - a.left;
  const int row_hi = p + a.right + 1 < lk ? p + a.right + 1 : lk;

  // Q and dO of the row, and delta = rowsum(dO * O).
  u32x4 qb[NS], dob[NS];
  float delta = 0.0f, nl = -__builtin_inf();
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int64_t at = (qi * a.hq + hh) * D + i * 16 + hb * 8;
    u32x4 ob = u32x4{0u, 0u, 0u, 0u};
    qb[i] = dob[i] = ob;
    if (row_ok) {
      qb[i] = *reinterpret_cast<const u32x4*>(a.q + qi * a.q_stride + (int64_t)hh * D + i * 16 +
                                              hb * 8);
      dob[i] = *reinterpret_cast<const u32x4*>(a.dout + at);
      ob = *reinterpret_cast<const u32x4*>(a.o + at);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      delta = __builtin_fmaf(to_f32<DT>((uint16_t)(dob[i][e] & 0xffffu)),
                             to_f32<DT>((uint16_t)(ob[e] & 0xffffu)), delta);
      delta = __builtin_fmaf(to_f32<DT>((uint16_t)(dob[i][e] >> 16)),
                             to_f32<DT>((uint16_t)(ob[e] >> 16)), delta);
    }
  }
  delta = half_sum(delta);
  if (row_ok) {
    const float lse = a.lse_in[(int64_t)hh * a.nq + qi];
    // exp2(x - LSE); a row that sees no key has LSE = -inf and P = 0
    nl = lse == -__builtin_inf() ? lse : -lse;
    if (lse == -__builtin_inf()) {
      delta = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) dob[i] = u32x4{0u, 0u, 0u, 0u};
    }
    if (hb == 0) {
      a.nlse[(int64_t)hh * a.nq + qi] = nl;
      a.delta[(int64_t)hh * a.nq + qi] = delta;
    }
  }
  TransposedRead<D> tr;
  tr.init(lane);

  const uint16_t* kh = a.k + (int64_t)s.k0 * a.k_stride + (int64_t)h * D;
  const uint16_t* vh = a.v + (int64_t)s.k0 * a.v_stride + (int64_t)h * D;
  auto tile_at = [&](int t, int* a0, int* cnt) __attribute__((always_inline)) {
    if (t < st) {
      *a0 = 0;
      *cnt = ns;
    } else {
      *a0 = lo + (t - st) * KT;
      *cnt = hi - *a0 < KT ? hi - *a0 : KT;
    }
  };
  auto load = [&](int t) __attribute__((always_inline)) {
    int a0, cnt;
    tile_at(t, &a0, &cnt);
    win_copy_tile<D, KT>(kh + (int64_t)a0 * a.k_stride, (uint32_t)a.k_stride * 2, cnt, sK[t & 1],
                         wv, lane);
    win_copy_tile<D, KT>(vh + (int64_t)a0 * a.v_stride, (uint32_t)a.v_stride * 2, cnt, sV[t & 1],
                         wv, lane);
  };
  const float* bias = nullptr;
  float *bins = nullptr, *skew = nullptr;
  float far_lo = 0.0f, far_hi = 0.0f;
  if constexpr (BIAS) {
    for (int i = 0; i < gt; ++i) win_load_bias<DT>(a, head0 + i, s_dyn + i * len, tid, 256);
    for (int i = tid; i < 4 * len; i += 256) s_bins[i] = 0.0f;
    for (int i = tid; i < 4 * SKEW_WORDS; i += 256) s_skew[i] = 0.0f;
    bias = s_dyn + (wv & gt_mask) * len;
    bins = s_bins + wv * len;
    skew = s_skew + wv * SKEW_WORDS;
  }

  f32x16 dq[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) dq[i][v] = 0.0f;

  if (nt > 0) load(0);
  for (int t = 0; t < nt; ++t) {
    wait_copies();
    __syncthreads();
    if (t + 1 < nt) load(t + 1);
    int a0, cnt;
    tile_at(t, &a0, &cnt);
    if (!wave_on || a0 >= w_hi || (a0 + cnt <= w_lo && a0 >= a.sinks)) continue;
    const char* ks = sK[t & 1];
    const char* vs = sV[t & 1];
    const bool edge =
        a0 + KT > (w_first + a.right + 1 < lk ? w_first + a.right + 1 : lk) ||
        a0 < w_last - a.left || cnt < KT;
    const int end = a0 + cnt < row_hi ? a0 + cnt : row_hi;
    const int c_hi = end - a0 - hb * 4, c_lo = row_lo - a0 - hb * 4,
              c_sink = a.sinks - a0 - hb * 4;
    const int rel_lo = a0 - w_last, rel_hi = a0 + KT - 1 - w_first;
    const bool far = BIAS && (rel_hi <= -a.range || rel_lo >= a.range);
    const bool far_right = rel_lo >= a.range;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      if (blk * 32 >= cnt) break;
      f32x16 sc, dp;
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = dp[v] = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int o = G::off(blk * 32 + l32, 2 * i + hb);
        sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(ks + o), qb[i], sc);
        dp = mfma32<DT>(*reinterpret_cast<const u32x4*>(vs + o), dob[i], dp);
      }
      float ds[16];
      const int off = BIAS ? WIN_PAD + a.range + a0 - p + hb * 4 : 0;
      if constexpr (BIAS) {
        if (far) {
          const float c = bias[WIN_PAD + (far_right ? 2 * a.range : 0)] + nl;
#pragma unroll
          for (int v = 0; v < 16; ++v)
            ds[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], a.scale_log2, c)) *
                    (dp[v] - delta);
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v)
            ds[v] = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(sc[v], a.scale_log2,
                                       bias[off + blk * 32 + acc_row(v, 0)]) + nl) *
                    (dp[v] - delta);
        }
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          ds[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], a.scale_log2, nl)) *
                  (dp[v] - delta);
      }
      if (edge) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = blk * 32 + acc_row(v, 0);
          if (!(c < c_hi && (c >= c_lo || c < c_sink))) ds[v] = 0.0f;
        }
      }
      if constexpr (BIAS) {
        if (far) {
          float sum = 0.0f;
#pragma unroll
          for (int v = 0; v < 16; ++v) sum += ds[v];
          if (far_right)
            far_hi += sum;
          else
            far_lo += sum;
        } else {
          float* put = skew + (hb * 4 + 31 - l32) * SKEW_PITCH + l32;
#pragma unroll
          for (int v = 0; v < 16; ++v) put[acc_row(v, 0) * SKEW_PITCH] = ds[v];
          wave_lds_order();
          if (lane < SKEW_ROWS) {
            const f32x4* row = reinterpret_cast<const f32x4*>(skew + lane * SKEW_PITCH);
            f32x4 sum = row[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) sum += row[i];
            bins[WIN_PAD + a.range + a0 + blk * 32 - w_first - 31 + lane] +=
                (sum[0] + sum[1]) + (sum[2] + sum[3]);
          }
          wave_lds_order();
        }
      }
      u32x4 db2[2];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          db2[c][e] = pack2<DT>(ds[c * 8 + 2 * e], ds[c * 8 + 2 * e + 1]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int db = 0; db < ND; ++db)
          dq[db] = mfma32<DT>(tr.read(ks, db, blk * 32 + c * 16), db2[c], dq[db]);
    }
  }

  if (row_ok) {
    uint16_t* orow = a.out + (qi * a.hq + hh) * D;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const int v = gi * 4;
        *reinterpret_cast<u32x2*>(orow + db * 32 + gi * 8 + hb * 4) =
            u32x2{pack2<DT>(dq[db][v] * a.scale, dq[db][v + 1] * a.scale),
                  pack2<DT>(dq[db][v + 2] * a.scale, dq[db][v + 3] * a.scale)};
      }
  }
  if constexpr (BIAS) {
    // the padding holds positions beyond the range
    static_assert(WIN_PAD == 96, "one and a half reads per lane");
    wave_lds_order();
    const float* above = bins + WIN_PAD + n_pos;
    far_lo += bins[lane];
    far_hi += above[lane];
    if (lane < 32) {
      far_lo += bins[64 + lane];
      far_hi += above[64 + lane];
    }
    for (int w = 32; w > 0; w >>= 1) {
      far_lo += __shfl_xor(far_lo, w);
      far_hi += __shfl_xor(far_hi, w);
    }
    if (lane == 0) bins[WIN_PAD] += far_lo;
    if (lane == 32 && a.range > 0) bins[WIN_PAD + 2 * a.range] += far_hi;
    // range 0: one position takes both sides
    wave_lds_order();
    if (a.range == 0 && lane == 32) bins[WIN_PAD] += far_hi;
    __syncthreads();
    for (int i = tid; i < gt * n_pos; i += 256) {
      const int hd = i / n_pos, m = i % n_pos;
      float sum = 0.0f;
      for (int w = hd; w < 4; w += gt) sum += s_bins[w * len + WIN_PAD + m];
      a.bias_part[((int64_t)tile * a.hq + head0) * n_pos + i] = sum;
    }
  }
}

// dK and dV of 128 keys of one kv head, each wave 32 of them, over the queries
// whose window holds them, head by head.  SINK: instead the partial sums of a
// sequence's first tokens over the queries of one chunk whose windows lie
// behind them.
template <int DT, int D, bool BIAS, bool SINK>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 128 ? 1 : 2, 2))) void
window_dkdv_kernel(WinArgs a) {
  using G = KvTile<D>;
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ __align__(1024) char sQ[2][G::BYTES];
  __shared__ __align__(1024) char sO[2][G::BYTES];
  __shared__ __align__(16) float s_nl[2][KT];
  __shared__ __align__(16) float s_delta[2][KT];
  extern __shared__ float s_bias[];

  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
  const int hb = lane >> 5, l32 = lane & 31;
  const int item = win_item();
  const int tiles = SINK ? a.n_sink_chunks : a.n_key_tiles;
  if (item >= tiles * (SINK ? a.hq : a.hkv)) return;
  // SINK: one query head at a time, else all of a kv head in turn
  const int head0 = SINK ? item / tiles : item / tiles * a.g, heads = SINK ? 1 : a.g;
  const int h = SINK ? head0 / a.g : item / tiles, tile = item % tiles;
  int idx;
  WinSeq s;
  if constexpr (SINK)
    s = win_sequence(a, win_find(a.cu_q, a.batch, a.nq, WIN_SINK_QUERIES, tile, &idx));
  else
    s = win_sequence(a, win_find(a.cu_k, a.batch, a.nk, WIN_KEYS, tile, &idx));
  if (s.b >= a.batch) s.lq = 0;  // keys behind the last sequence: zero gradients
  const int pos_min = s.lk - s.lq;  // position of query 0
  int j0, kn, i_lo, i_hi;           // keys j0 .. j0 + kn - 1, queries i_lo .. i_hi - 1
  if constexpr (SINK) {
    if (idx < 0 || (int64_t)idx * WIN_SINK_QUERIES >= s.lq) return;
    j0 = 0;
    kn = a.sinks < s.lk ? a.sinks : s.lk;
    i_lo = idx * WIN_SINK_QUERIES;
    i_hi = i_lo + WIN_SINK_QUERIES < s.lq ? i_lo + WIN_SINK_QUERIES : s.lq;
    const int first = a.left + 1 - pos_min;  // key 0 has left the window here
    if (i_lo < first) i_lo = first < i_hi ? first : i_hi;
    if (kn <= 0) i_lo = i_hi;
  } else {
    if (idx < 0 || (int64_t)idx * WIN_KEYS >= s.lk) return;
    j0 = idx * WIN_KEYS;
    kn = s.lk - j0 < WIN_KEYS ? s.lk - j0 : WIN_KEYS;
    i_lo = j0 - a.right - pos_min;
    i_lo = i_lo > 0 ? i_lo : 0;
    i_hi = j0 + kn - pos_min + a.left;
    i_hi = i_hi < s.lq ? i_hi : s.lq;
  }
  const int ntq = i_hi > i_lo ? (i_hi - i_lo + KT - 1) / KT : 0;
  const int steps = ntq * heads;

  // This wave's keys, as B operands.
  const int jw = j0 + wv * 32, j = jw + l32;
  const bool key_ok = wv * 32 + l32 < kn;
  const bool wave_on = wv * 32 < kn;
  u32x4 kb[NS], vb[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    kb[i] = vb[i] = u32x4{0u, 0u, 0u, 0u};
    if (key_ok) {
      const int64_t c = (int64_t)h * D + i * 16 + hb * 8;
      kb[i] = *reinterpret_cast<const u32x4*>(a.k + (int64_t)(s.k0 + j) * a.k_stride + c);
      vb[i] = *reinterpret_cast<const u32x4*>(a.v + (int64_t)(s.k0 + j) * a.v_stride + c);
    }
  }
  TransposedRead<D> tr;
  tr.init(lane);

  auto load = [&](int step) __attribute__((always_inline)) {
    const int hh = head0 + step / ntq, i = i_lo + (step % ntq) * KT;
    const int cnt = i_hi - i < KT ? i_hi - i : KT;
    const int64_t qi = (int64_t)s.q0 + i;
    const int b = step & 1;
    win_copy_tile<D, KT>(a.q + qi * a.q_stride + (int64_t)hh * D, (uint32_t)a.q_stride * 2, cnt,
                         sQ[b], wv, lane);
    win_copy_tile<D, KT>(a.dout + (qi * a.hq + hh) * D, (uint32_t)a.hq * D * 2, cnt, sO[b], wv,
                         lane);
    if (wv == 0) win_copy_floats(a.nlse + (int64_t)hh * a.nq + qi, cnt, s_nl[b], lane);
    if (wv == 1) win_copy_floats(a.delta + (int64_t)hh * a.nq + qi, cnt, s_delta[b], lane);
  };

  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) dk[i][v] = dv[i][v] = 0.0f;

  if (steps > 0) load(0);
  for (int step = 0; step < steps; ++step) {
    wait_copies();
    __syncthreads();
    if (step + 1 < steps) load(step + 1);
    if constexpr (BIAS) {
      if (step % ntq == 0) {
        win_load_bias<DT>(a, head0 + step / ntq, s_bias, tid, 256);
        __syncthreads();
      }
    }
    const int i = i_lo + (step % ntq) * KT;
    const int cnt = i_hi - i < KT ? i_hi - i : KT;
    if (!wave_on) continue;
    const char* qs = sQ[step & 1];
    const char* os = sO[step & 1];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int p0 = pos_min + i + rb * 32, p1 = p0 + 31;  // positions of the rows
      if (rb * 32 >= cnt) break;
      if constexpr (SINK) {
        if (p1 <= jw + a.left) continue;
      } else {
        if (jw > p1 + a.right || jw + 31 < p0 - a.left) continue;
      }
      f32x16 sc, dp;
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = dp[v] = 0.0f;
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int o = G::off(rb * 32 + l32, 2 * x + hb);
        sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(qs + o), kb[x], sc);
        dp = mfma32<DT>(*reinterpret_cast<const u32x4*>(os + o), vb[x], dp);
      }
      float pr[16], ds[16];
      f32x4 nl[4], dl[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        nl[x] = *reinterpret_cast<const f32x4*>(&s_nl[step & 1][rb * 32 + x * 8 + hb * 4]);
        dl[x] = *reinterpret_cast<const f32x4*>(&s_delta[step & 1][rb * 32 + x * 8 + hb * 4]);
      }
      if constexpr (BIAS) {
        const int rel_lo = jw - p1, rel_hi = jw + 31 - p0;
        if (rel_hi <= -a.range || rel_lo >= a.range) {
          const float c = s_bias[WIN_PAD + (rel_lo >= a.range ? 2 * a.range : 0)];
#pragma unroll
          for (int v = 0; v < 16; ++v)
            pr[v] = __builtin_amdgcn_exp2f(
                __builtin_fmaf(sc[v], a.scale_log2, c + nl[v / 4][v % 4]));
        } else {
          const float* at = s_bias + WIN_PAD + a.range + j - p0 - hb * 4 - 31;
#pragma unroll
          for (int v = 0; v < 16; ++v)
            pr[v] = __builtin_amdgcn_exp2f(
                __builtin_fmaf(sc[v], a.scale_log2, at[31 - acc_row(v, 0)]) + nl[v / 4][v % 4]);
        }
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          pr[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], a.scale_log2, nl[v / 4][v % 4]));
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) ds[v] = pr[v] * (dp[v] - dl[v / 4][v % 4]);
      bool edge;
      if constexpr (SINK)
        edge = true;
      else
        edge = jw + 31 > p0 + a.right || jw < p1 - a.left || rb * 32 + 32 > cnt;
      if (edge) {
        // rows c .. of this lane's half, as offsets from p0 + 4 hb
        const int base = p0 + hb * 4;
        int c_lo, c_hi = cnt - rb * 32 - hb * 4;
        if constexpr (SINK) {
          c_lo = j + a.left + 1 - base;
          if (j >= a.sinks) c_hi = 0;
        } else {
          c_lo = j - a.right - base;
          const int c = j + a.left + 1 - base;
          c_hi = c < c_hi ? c : c_hi;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = acc_row(v, 0);
          if (!(c >= c_lo && c < c_hi)) pr[v] = ds[v] = 0.0f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u32x4 pb, db2;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pb[e] = pack2<DT>(pr[c * 8 + 2 * e], pr[c * 8 + 2 * e + 1]);
          db2[e] = pack2<DT>(ds[c * 8 + 2 * e], ds[c * 8 + 2 * e + 1]);
        }
#pragma unroll
        for (int db = 0; db < ND; ++db) {
          dv[db] = mfma32<DT>(tr.read(os, db, rb * 32 + c * 16), pb, dv[db]);
          dk[db] = mfma32<DT>(tr.read(qs, db, rb * 32 + c * 16), db2, dk[db]);
        }
      }
    }
  }

  if constexpr (SINK) {
    if (wv * 32 + l32 < a.sinks) {
      float* out = a.sink_part +
                   (((int64_t)tile * a.hq + head0) * 2 * a.sinks + wv * 32 + l32) * D;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          out[db * 32 + acc_row(v, hb)] = dk[db][v];
          out[(int64_t)a.sinks * D + db * 32 + acc_row(v, hb)] = dv[db][v];
        }
    }
  } else {
    if (!key_ok) return;
    if (a.sink_sum && j < a.sinks && s.b < a.batch) {
      const float* add = a.sink_sum + (((int64_t)s.b * a.hkv + h) * 2 * a.sinks + j) * D;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          dk[db][v] += add[db * 32 + acc_row(v, hb)];
          dv[db][v] += add[(int64_t)a.sinks * D + db * 32 + acc_row(v, hb)];
        }
    }
    const int64_t row = ((int64_t)(s.k0 + j) * a.hkv + h) * D;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const int v = gi * 4;
        const int64_t at = row + db * 32 + gi * 8 + hb * 4;
        *reinterpret_cast<u32x2*>(a.dk + at) =
            u32x2{pack2<DT>(dk[db][v] * a.scale, dk[db][v + 1] * a.scale),
                  pack2<DT>(dk[db][v + 2] * a.scale, dk[db][v + 3] * a.scale)};
        *reinterpret_cast<u32x2*>(a.dv + at) = u32x2{pack2<DT>(dv[db][v], dv[db][v + 1]),
                                                     pack2<DT>(dv[db][v + 2], dv[db][v + 3])};
      }
  }
}

// sink_sum of one sequence and kv head, 64 words a workgroup: 16 waves take
// every 16th of its partial sums (chunk by chunk, head by head), and their sums
// are added in wave order.
__global__ __launch_bounds__(1024) void window_sink_sum_kernel(WinArgs a, int d) {
  __shared__ float part[16][64];
  const int lane = lane_id(), wv = wave_id();
  const int b = blockIdx.x / a.hkv, h = blockIdx.x % a.hkv;
  const WinSeq s = win_sequence(a, b);
  const int first = win_offset(a.cu_q, b, a.nq) / WIN_SINK_QUERIES + b;
  int n = (s.lq + WIN_SINK_QUERIES - 1) / WIN_SINK_QUERIES;
  if (n > a.n_sink_chunks - first) n = a.n_sink_chunks - first;
  const int words = 2 * a.sinks * d, e = blockIdx.y * 64 + lane;  // words: a multiple of 64
  float sum = 0.0f;
  for (int x = wv; x < n * a.g; x += 16)
    sum += a.sink_part[((int64_t)(first + x / a.g) * a.hq + h * a.g + x % a.g) * words + e];
  part[wv][lane] = sum;
  __syncthreads();
  if (wv == 0) {
    for (int w = 1; w < 16; ++w) sum += part[w][lane];
    a.sink_sum[((int64_t)b * a.hkv + h) * words + e] = sum;
  }
}

// Sums of dS per position over the query tiles: 16 waves take every 16th
// tile, 64 positions of one head, and their sums are added in wave order.
__global__ __launch_bounds__(1024) void window_bias_sum_kernel(WinArgs a) {
  __shared__ float part[16][64];
  const int n_pos = 2 * a.range + 1, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int head = blockIdx.x, m = blockIdx.y * 64 + lane;
  float sum = 0.0f;
  if (m < n_pos)
    for (int t = wv; t < a.n_tiles; t += 16)
      sum += a.bias_part[((int64_t)t * a.hq + head) * n_pos + m];
  part[wv][lane] = sum;
  __syncthreads();
  if (wv == 0 && m < n_pos) {
    for (int w = 1; w < 16; ++w) sum += part[w][lane];
    a.bias_sum[head * n_pos + m] = sum;
  }
}

// Gradient of the table, rounded once: a wave per (bucket, head), every lane
// every 64th position of the bucket.
template <int DT>
__global__ __launch_bounds__(256) void window_bias_table_kernel(WinArgs a) {
  const int n_pos = 2 * a.range + 1, lane = lane_id();
  const int64_t t = (int64_t)blockIdx.x * 4 + wave_id();
  if (t >= (int64_t)a.n_buckets * a.hq) return;
  const int b = (int)(t / a.hq), head = (int)(t % a.hq);
  float sum = 0.0f;
  for (int m = lane; m < n_pos; m += 64) {
    int x = a.buckets[m];
    x = x < 0 ? 0 : (x >= a.n_buckets ? a.n_buckets - 1 : x);
    if (x == b) sum += a.bias_sum[head * n_pos + m];
  }
  for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
  if (lane == 0) a.dtable[t] = from_f32<DT>(sum);
}

struct WinBwdWs {
  float *nlse, *delta, *sink_part, *sink_sum, *bias_part, *bias_sum;
};

// Whether any query may have left the first tokens behind its window.
static bool has_sinks(int64_t nk, int64_t left, int64_t sinks) {
  return sinks > 0 && left >= 0 && left < nk - 1;
}

static void carve(Carver& c, WinBwdWs& w, int64_t nq, int64_t nk, int64_t hq, int64_t hkv,
                  int64_t d, int64_t batch, int64_t left, int64_t sinks, int64_t range) {
  w = WinBwdWs{};
  w.nlse = c.take<float>((size_t)(nq * hq));
  w.delta = c.take<float>((size_t)(nq * hq));
  if (has_sinks(nk, left, sinks)) {
    w.sink_part = c.take<float>((size_t)win_tiles(nq, WIN_SINK_QUERIES, batch) * hq * 2 * sinks *
                                d);
    w.sink_sum = c.take<float>((size_t)batch * hkv * 2 * sinks * d);
  }
  if (range >= 0) {
    const int64_t g = hq / hkv, tq = g % 4 == 0 ? 32 : (g % 2 == 0 ? 64 : 128);
    w.bias_part = c.take<float>((size_t)win_tiles(nq, tq, batch) * hq * (2 * range + 1));
    w.bias_sum = c.take<float>((size_t)hq * (2 * range + 1));
  }
}

template <int DT, int D, bool BIAS>
static int bwd_launch(const WinArgs& a, hipStream_t st) {
  const size_t bias_lds = BIAS ? (size_t)win_bias_len(a.range) * 4 : 0;
  const dim3 block(256);
  if (a.nq > 0 || BIAS) {  // (every tile's sums of dS are read)
    hipLaunchKernelGGL((window_dq_kernel<DT, D, BIAS>),
                       dim3(win_grid((int64_t)a.n_tiles * a.hkv * (a.g >> a.gt_log2))), block,
                       BIAS ? bias_lds * (4 + (1 << a.gt_log2)) + 16 * SKEW_WORDS + 16 : 0, st, a);
    LSRM_CHECK_LAUNCH();
  }
  if (a.nk > 0) {
    if (a.sink_part) {
      hipLaunchKernelGGL((window_dkdv_kernel<DT, D, BIAS, true>),
                         dim3(win_grid((int64_t)a.n_sink_chunks * a.hq)), block, bias_lds, st,
                         a);
      LSRM_CHECK_LAUNCH();
      if (a.batch > 0) {
        hipLaunchKernelGGL(window_sink_sum_kernel, dim3(a.batch * a.hkv, 2 * a.sinks * D / 64),
                           dim3(1024), 0, st, a, D);
        LSRM_CHECK_LAUNCH();
      }
    }
    hipLaunchKernelGGL((window_dkdv_kernel<DT, D, BIAS, false>),
                       dim3(win_grid((int64_t)a.n_key_tiles * a.hkv)), block, bias_lds, st, a);
    LSRM_CHECK_LAUNCH();
  }
  if constexpr (BIAS) {
    hipLaunchKernelGGL(window_bias_sum_kernel, dim3(a.hq, ceil_div(2 * a.range + 1, 64)),
                       dim3(1024), 0, st, a);
    LSRM_CHECK_LAUNCH();
    hipLaunchKernelGGL(window_bias_table_kernel<DT>,
                       dim3(ceil_div((int64_t)a.n_buckets * a.hq, 4)), block, 0, st, a);
    LSRM_CHECK_LAUNCH();
  }
  return LSRM_OK;
}

template <int DT>
static int bwd_dims(const WinArgs& a, int64_t d, hipStream_t st) {
  if (a.table) {
    if (d == 32) return bwd_launch<DT, 32, true>(a, st);
    if (d == 64) return bwd_launch<DT, 64, true>(a, st);
    return bwd_launch<DT, 128, true>(a, st);
  }
  if (d == 32) return bwd_launch<DT, 32, false>(a, st);
  if (d == 64) return bwd_launch<DT, 64, false>(a, st);
  return bwd_launch<DT, 128, false>(a, st);
}

}  // namespace lsrm

using namespace lsrm;

extern "C" size_t lsrm_window_attn_bwd_workspace_size(int64_t n_q, int64_t n_k, int64_t hq,
                                                      int64_t hkv, int64_t head_dim,
                                                      int64_t batch, int64_t left, int64_t sinks,
                                                      int64_t bias_range) {
  if (n_q < 0 || n_k < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || head_dim <= 0 || batch < 0 ||
      sinks < 0 || sinks > WIN_MAX_SINKS || bias_range > WIN_MAX_RANGE || n_q > WIN_MAX_TOKENS ||
      n_k > WIN_MAX_TOKENS || batch > WIN_MAX_TOKENS)
    return 0;
  Carver c{nullptr, 0, 0};
  WinBwdWs w;
  carve(c, w, n_q, n_k, hq, hkv, head_dim, batch, left, sinks, bias_range);
  return c.used + 256;
}

extern "C" int lsrm_window_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                                    const void* o, const float* lse, int dtype, int64_t q_stride,
                                    int64_t k_stride, int64_t v_stride, int64_t n_q, int64_t n_k,
                                    int64_t hq, int64_t hkv, int64_t head_dim,
                                    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                    int64_t batch, int64_t left, int64_t right, int64_t sinks,
                                    const void* bias_table, int64_t n_buckets,
                                    const int32_t* bias_buckets, int64_t bias_range,
                                    float softmax_scale, void* dq, void* dk, void* dv,
                                    void* d_table, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  WinArgs a;
  const int rc = win_args(a, q, k, v, dtype, q_stride, k_stride, v_stride, n_q, n_k, hq, hkv,
                          head_dim, cu_seqlens_q, cu_seqlens_k, batch, left, right, sinks,
                          bias_table, n_buckets, bias_buckets, bias_range, softmax_scale);
  if (rc) return rc;
  if ((n_q > 0 && (!dout || !o || !lse || !dq)) || (n_k > 0 && (!dk || !dv)) ||
      (bias_table != nullptr) != (d_table != nullptr))
    return LSRM_ERR_INVALID_ARG;
  if (((uintptr_t)dout | (uintptr_t)o | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15u)
    return LSRM_ERR_UNSUPPORTED;
  if (hq * head_dim > WIN_MAX_STRIDE) return LSRM_ERR_UNSUPPORTED;
  Carver c{(char*)workspace, 0, workspace_bytes};
  WinBwdWs w;
  carve(c, w, n_q, n_k, hq, hkv, head_dim, batch, left, sinks, bias_table ? bias_range : -1);
  if (!workspace || !c.ok()) return LSRM_ERR_WORKSPACE;
  a.dout = (const uint16_t*)dout;
  a.o = (const uint16_t*)o;
  a.lse_in = lse;
  a.out = (uint16_t*)dq;
  a.dk = (uint16_t*)dk;
  a.dv = (uint16_t*)dv;
  a.nlse = w.nlse;
  a.delta = w.delta;
  a.sink_part = w.sink_part;
  a.sink_sum = w.sink_sum;
  a.bias_part = w.bias_part;
  a.bias_sum = w.bias_sum;
  a.dtable = (uint16_t*)d_table;
  a.n_key_tiles = win_tiles(n_k, WIN_KEYS, batch);
  a.n_sink_chunks = win_tiles(n_q, WIN_SINK_QUERIES, batch);
  if ((int64_t)a.n_key_tiles * hkv > INT32_MAX - NXCD ||
      (int64_t)a.n_sink_chunks * hq > INT32_MAX - NXCD || batch * hkv > INT32_MAX)
    return LSRM_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  return dtype == LSRM_BF16 ? bwd_dims<LSRM_BF16>(a, head_dim, st)
                            : bwd_dims<LSRM_F16>(a, head_dim, st);
}
