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
//
// Both are bound like the forward, by matrix and vector instructions in turn: 32
// by 32 elements at head dim 64 are 384 cycles of MFMA and 420 of vector work
// for dQ (960 taken), 512 and 420 for dK/dV (1330 taken, two waves a SIMD and
// whole waves that see nothing at both ends of a tile's queries).  32768 tokens,
// 16 heads of 64, windows of 1024: dQ 253 us, 800 TFLOP/s, dK/dV 336 us, 805; 8
// heads of 128: 248 us, 820, and 473 us, 570 (one wave a SIMD).  Tried without
// gain: two row blocks at once (7% more time), three waves a SIMD (spills), rows
// read ahead of the exponentials, dS rows that wait for the next block.
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
// 979 us at 32768 tokens, 16 heads of 64, windows of 511, R = 128; this way 283,
// and 179 without a bias.)
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
  const int w_all = w_first + a.right + 1 < lk ? w_first + a.right + 1 : lk;
  const int p = w_first + l32;
  const int row_lo = p - a.left;
  const int row_hi = p + a.right + 1 < lk ? p + a.right + 1 : lk;

  const uint16_t* kh = a.k + (int64_t)s.k0 * a.k_stride + (int64_t)h * D;
  const uint16_t* vh = a.v + (int64_t)s.k0 * a.v_stride + (int64_t)h * D;
  TileCopy<D, KT> kc, vc;
  kc.init(a.k_stride, wv, lane);
  vc.init(a.v_stride, wv, lane);
  auto tile_at = [&](int t, int* a0, int* cnt) __attribute__((always_inline)) {
    *a0 = t < st ? 0 : lo + (t - st) * KT;
    const int end = t < st ? ns : hi;
    *cnt = end - *a0 < KT ? end - *a0 : KT;
  };
  auto load = [&](int t) __attribute__((always_inline)) {
    int a0, cnt;
    tile_at(t, &a0, &cnt);
    kc.copy(kh + (int64_t)a0 * a.k_stride, cnt, sK[t & 1], wv, lane);
    vc.copy(vh + (int64_t)a0 * a.v_stride, cnt, sV[t & 1], wv, lane);
  };
  if (nt > 0) load(0);  // in flight while the rest is read

  // Q and dO of the row, and delta = rowsum(dO * O).
  u32x4 qb[NS], dob[NS];
  float delta = 0.0f, nl = -__builtin_inf();
  u32x4 low[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    low[i] = u32x4{0u, 0u, 0u, 0u};
    if (row_ok && a.o_low)
      low[i] = reinterpret_cast<const u32x4*>(a.o_low + (qi * a.hq + hh) * D + hb * (D / 2))[i];
  }
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
      const int l = (int)(low[i / 2][(i % 2) * 2 + e / 2] >> (16 * (e % 2)));  // two bytes
      delta = __builtin_fmaf(to_f32<DT>((uint16_t)(dob[i][e] & 0xffffu)),
                             with_low<DT>((uint16_t)(ob[e] & 0xffffu), (int8_t)l), delta);
      delta = __builtin_fmaf(to_f32<DT>((uint16_t)(dob[i][e] >> 16)),
                             with_low<DT>((uint16_t)(ob[e] >> 16), (int8_t)(l >> 8)), delta);
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
      a.ndelta[(int64_t)hh * a.nq + qi] = -delta;
    }
  }
  f32x16 nd;
#pragma unroll
  for (int v = 0; v < 16; ++v) nd[v] = -delta;
  TransposedRead<D> tr;
  tr.init(lane);

  const float* bias = nullptr;
  float *bins = nullptr, *skew = nullptr;
  float far_lo = 0.0f, far_hi = 0.0f;
  if constexpr (BIAS) {
    win_load_bias<DT>(a, head0, gt, s_dyn, tid);
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

  for (int t = 0; t < nt; ++t) {
    wait_copies();
    __syncthreads();
    if (t + 1 < nt) load(t + 1);
    int a0, cnt;
    tile_at(t, &a0, &cnt);
    if (!wave_on || a0 >= w_hi || (a0 + cnt <= w_lo && a0 >= a.sinks)) continue;
    const char* ks = sK[t & 1];
    const char* vs = sV[t & 1];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int k0 = a0 + blk * 32;  // first key of the block
      if (blk * 32 >= cnt || k0 >= w_hi || (k0 + 32 <= w_lo && k0 >= a.sinks)) continue;
      const bool edge = k0 + 32 > w_all || k0 < w_last - a.left || blk * 32 + 32 > cnt;
      const int rel_lo = k0 - w_last, rel_hi = k0 + 31 - w_first;
      const bool far = BIAS && (rel_hi <= -a.range || rel_lo >= a.range);
      const bool far_right = rel_lo >= a.range;
      f32x16 sc, dp = nd;  // dP - delta
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
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
            ds[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], a.scale_log2, c)) * dp[v];
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v)
            ds[v] = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(sc[v], a.scale_log2,
                                       bias[off + blk * 32 + acc_row(v, 0)]) + nl) *
                    dp[v];
        }
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          ds[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[v], a.scale_log2, nl)) * dp[v];
      }
      if (edge) {
        const int end = a0 + cnt < row_hi ? a0 + cnt : row_hi, base = k0 + hb * 4;
        const uint32_t seen = bits_below(end - base) &
                              (~bits_below(row_lo - base) | bits_below(a.sinks - base));
#pragma unroll
        for (int v = 0; v < 16; ++v) ds[v] = keep(seen, v, ds[v], 0.0f);
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

  uint16_t* orow = a.out + (qi * a.hq + hh) * D + hb * 8;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const u32x4 piece = row_piece<DT>(dq[i / 2], i % 2, a.scale);
    if (row_ok) *reinterpret_cast<u32x4*>(orow + i * 16) = piece;
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
// whose window holds them, 64 at a time, head by head.  With few keys the heads
// of a group are split between `head_splits` workgroups, whose fp32 sums
// window_dkdv_join_kernel adds.
// SINK: instead the partial sums of 32 of a sequence's first tokens over the
// queries of one chunk and head whose windows lie behind them, 128 at a time,
// each wave 32 of them; the waves' sums are added in LDS in wave order.
template <int DT, int D, bool BIAS, bool SINK>
__global__ __launch_bounds__(256)
    __attribute__((amdgpu_waves_per_eu(D == 128 ? 1 : (D == 32 ? 3 : 2), 4))) void
window_dkdv_kernel(WinArgs a) {
  constexpr int NR = SINK ? 128 : KT;  // query rows per step
  using G = KvTile<D, NR>;
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ __align__(1024) char s_rows[2][2][G::BYTES];  // Q / dO, buffer
  __shared__ __align__(16) float s_nl[2][NR];
  __shared__ __align__(16) float s_nd[2][NR];
  extern __shared__ float s_bias[];

  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
  const int hb = lane >> 5, l32 = lane & 31;
  const int item = win_item();
  // SINK: chunk, head, 32 of the first tokens; else key tile, kv head, part of
  // its query heads.
  const int tiles = SINK ? a.n_sink_chunks : a.n_key_tiles;
  const int tile = item % tiles, rest = item / tiles;
  const int minor = SINK ? (a.sinks + 31) / 32 : a.head_splits;
  if (rest >= (SINK ? a.hq : a.hkv) * minor) return;
  const int part = rest % minor;
  const int per = (a.g + a.head_splits - 1) / a.head_splits;
  const int h = SINK ? rest / minor / a.g : rest / minor;
  const int head0 = SINK ? rest / minor : h * a.g + part * per;
  const int heads = SINK ? 1 : (a.g - part * per < per ? a.g - part * per : per);
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
    j0 = part * 32;
    kn = (a.sinks < s.lk ? a.sinks : s.lk) - j0;
    i_lo = idx * WIN_SINK_QUERIES;
    i_hi = i_lo + WIN_SINK_QUERIES < s.lq ? i_lo + WIN_SINK_QUERIES : s.lq;
    const int first = j0 + a.left + 1 - pos_min;  // key j0 has left the window here
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
  const int ntq = i_hi > i_lo ? (i_hi - i_lo + NR - 1) / NR : 0;
  const int steps = heads > 0 ? ntq * heads : 0;

  TransposedRead<D> tr;
  tr.init(lane);
  TileCopy<D, NR> qc, oc;
  qc.init(a.q_stride, wv, lane);
  oc.init((int64_t)a.hq * D, wv, lane);

  int ld_head = head0, ld_i = i_lo;  // of the next step to load
  auto load = [&](int b) __attribute__((always_inline)) {
    const int cnt = i_hi - ld_i < NR ? i_hi - ld_i : NR;
    const int64_t qi = (int64_t)s.q0 + ld_i;
    qc.copy(a.q + qi * a.q_stride + (int64_t)ld_head * D, cnt, s_rows[0][b], wv, lane);
    oc.copy(a.dout + (qi * a.hq + ld_head) * D, cnt, s_rows[1][b], wv, lane);
    const int w64 = (wv >> 1) * 64;  // two waves per 64 rows
    if (w64 < NR) {
      const int from = w64 < cnt ? w64 : cnt - 1, left = w64 < cnt ? cnt - w64 : 1;
      const float* src = (wv & 1 ? a.ndelta : a.nlse) + (int64_t)ld_head * a.nq + qi + from;
      win_copy_floats(src, left, (wv & 1 ? s_nd[b] : s_nl[b]) + w64, lane);
    }
    ld_i += NR;
    if (ld_i >= i_hi) {
      ld_i = i_lo;
      ++ld_head;
    }
  };
  if (steps > 0) load(0);  // in flight while the keys are read

  // This wave's keys, as B operands.
  const int jw = j0 + (SINK ? 0 : wv * 32), j = jw + l32;
  const bool key_ok = j < j0 + kn;
  const bool wave_on = jw < j0 + kn;
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
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) dk[i][v] = dv[i][v] = 0.0f;

  int head = head0, i = i_lo;
  for (int step = 0; step < steps; ++step) {
    wait_copies();
    __syncthreads();
    if (step + 1 < steps) load((step + 1) & 1);
    if constexpr (BIAS) {
      if (i == i_lo) {
        win_load_bias<DT>(a, head, 1, s_bias, tid);
        __syncthreads();
      }
    }
    const int cnt = i_hi - i < NR ? i_hi - i : NR;
    const char* qs = s_rows[0][step & 1];
    const char* os = s_rows[1][step & 1];
#pragma unroll
    for (int rr = 0; rr < (SINK ? 1 : 2); ++rr) {
      const int rb = SINK ? wv : rr;
      const int p0 = pos_min + i + rb * 32, p1 = p0 + 31;  // positions of the rows
      if (!wave_on || rb * 32 >= cnt) continue;
      if constexpr (SINK) {
        if (p1 <= jw + a.left) continue;
      } else {
        if (jw > p1 + a.right || jw + 31 < p0 - a.left) continue;
      }
      f32x16 sc, dp;
      f32x4 nl[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = rb * 32 + x * 8 + hb * 4;
        if constexpr (D == 128) nl[x] = *reinterpret_cast<const f32x4*>(&s_nl[step & 1][row]);
        const f32x4 t = *reinterpret_cast<const f32x4*>(&s_nd[step & 1][row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[x * 4 + e] = t[e];  // dP - delta
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int o = rb * 32 * (D * 2) + G::off(l32, 2 * x + hb);
        sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(qs + o), kb[x], sc);
        dp = mfma32<DT>(*reinterpret_cast<const u32x4*>(os + o), vb[x], dp);
      }
      // At head dims 32 and 64 nothing below is read ahead of the products: fewer
      // registers, 2% less time.  At 128, with one wave per SIMD, the rows' numbers
      // are read before them: later they cost spills, and 25% more time.
      if constexpr (D <= 64) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          nl[x] = *reinterpret_cast<const f32x4*>(&s_nl[step & 1][rb * 32 + x * 8 + hb * 4]);
      }
      float pr[16], ds[16];
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
      for (int v = 0; v < 16; ++v) ds[v] = pr[v] * dp[v];
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
        const uint32_t seen = bits_between(c_lo, c_hi);
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          pr[v] = keep(seen, v, pr[v], 0.0f);
          ds[v] = keep(seen, v, ds[v], 0.0f);
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
    i += NR;
    if (i >= i_hi) {
      i = i_lo;
      ++head;
    }
  }

  if constexpr (SINK) {
    constexpr int RED = 2 * ND * 16;
    static_assert(3 * RED * 64 * 4 <= 4 * G::BYTES, "the waves' sums fit where the rows were");
    __syncthreads();
    float* red = reinterpret_cast<float*>(&s_rows[0][0][0]) + lane;
    if (wv > 0) {
      float* mine = red + (wv - 1) * RED * 64;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          mine[(db * 16 + v) * 64] = dk[db][v];
          mine[((ND + db) * 16 + v) * 64] = dv[db][v];
        }
    }
    __syncthreads();
    if (wv > 0 || j >= a.sinks) return;
    float* out = a.sink_part + (((int64_t)tile * a.hq + head0) * 2 * a.sinks + j) * D;
#pragma unroll 1
    for (int w = 0; w < 3; ++w, red += RED * 64)
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          dk[db][v] += red[(db * 16 + v) * 64];
          dv[db][v] += red[((ND + db) * 16 + v) * 64];
        }
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        out[db * 32 + acc_row(v, hb)] = dk[db][v];
        out[(int64_t)a.sinks * D + db * 32 + acc_row(v, hb)] = dv[db][v];
      }
  } else {
    if (a.head_splits > 1) {
      if (!key_ok) return;
      // [part, key, kv head, dK / dV, d]
      float* out = a.head_part + (((int64_t)part * a.nk + s.k0 + j) * a.hkv + h) * 2 * D;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int gi = 0; gi < 4; ++gi) {
          const int v = gi * 4, at = db * 32 + gi * 8 + hb * 4;
          *reinterpret_cast<f32x4*>(out + at) =
              f32x4{dk[db][v], dk[db][v + 1], dk[db][v + 2], dk[db][v + 3]};
          *reinterpret_cast<f32x4*>(out + D + at) =
              f32x4{dv[db][v], dv[db][v + 1], dv[db][v + 2], dv[db][v + 3]};
        }
      return;
    }
    if (key_ok && a.sink_sum && j < a.sinks && s.b < a.batch) {
      const float* add = a.sink_sum + (((int64_t)s.b * a.hkv + h) * 2 * a.sinks + j) * D;
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          dk[db][v] += add[db * 32 + acc_row(v, hb)];
          dv[db][v] += add[(int64_t)a.sinks * D + db * 32 + acc_row(v, hb)];
        }
    }
    const int64_t row = ((int64_t)(s.k0 + j) * a.hkv + h) * D + hb * 8;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const u32x4 kp = row_piece<DT>(dk[i / 2], i % 2, a.scale);
      const u32x4 vp = row_piece<DT>(dv[i / 2], i % 2, 1.0f);
      if (!key_ok) continue;
      *reinterpret_cast<u32x4*>(a.dk + row + i * 16) = kp;
      *reinterpret_cast<u32x4*>(a.dv + row + i * 16) = vp;
    }
  }
}

// dK and dV from the head parts' sums in order (and the first tokens' sums);
// one thread per four channels of a key.
template <int DT, int D>
__global__ __launch_bounds__(256) void window_dkdv_join_kernel(WinArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  constexpr int PER = 2 * D / 4;  // threads per (key, kv head)
  const int64_t row = t / PER;
  const int at = (int)(t % PER) * 4;  // channel of dK, then of dV
  if (row >= (int64_t)a.nk * a.hkv) return;
  f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
  for (int p = 0; p < a.head_splits; ++p)
    sum += *reinterpret_cast<const f32x4*>(a.head_part +
                                           ((int64_t)p * a.nk * a.hkv + row) * 2 * D + at);
  if (a.sink_sum) {
    const int key = (int)(row / a.hkv), h = (int)(row % a.hkv);
    int lo = 0, hi = a.batch;
    while (lo < hi) {  // largest sequence that begins at or before the key
      const int mid = (lo + hi + 1) >> 1;
      if (win_offset(a.cu_k, mid, a.nk) <= key)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int j = key - win_offset(a.cu_k, lo, a.nk);
    if (lo < a.batch && j >= 0 && j < a.sinks)
      sum += *reinterpret_cast<const f32x4*>(
          a.sink_sum + ((((int64_t)lo * a.hkv + h) * 2 + at / D) * a.sinks + j) * D + at % D);
  }
  uint16_t* out = (at < D ? a.dk : a.dv) + row * D + at % D;
  const float f = at < D ? a.scale : 1.0f;
  *reinterpret_cast<u32x2*>(out) =
      u32x2{pack2<DT>(sum[0] * f, sum[1] * f), pack2<DT>(sum[2] * f, sum[3] * f)};
}

// sink_sum of one sequence and kv head, 16 words a workgroup: 64 threads a
// word take every 64th of its partial sums (chunk by chunk, head by head), and
// their sums are added in order.
__global__ __launch_bounds__(1024) void window_sink_sum_kernel(WinArgs a, int d) {
  __shared__ float part[64][17];
  const int col = threadIdx.x & 15, at = threadIdx.x >> 4;
  const int b = blockIdx.x / a.hkv, h = blockIdx.x % a.hkv;
  const WinSeq s = win_sequence(a, b);
  const int first = win_offset(a.cu_q, b, a.nq) / WIN_SINK_QUERIES + b;
  int n = (s.lq + WIN_SINK_QUERIES - 1) / WIN_SINK_QUERIES;
  if (n > a.n_sink_chunks - first) n = a.n_sink_chunks - first;
  const int words = 2 * a.sinks * d, e = blockIdx.y * 16 + col;  // words: a multiple of 64
  float sum = 0.0f;
  for (int x = at; x < n * a.g; x += 64)
    sum += a.sink_part[((int64_t)(first + x / a.g) * a.hq + h * a.g + x % a.g) * words + e];
  part[at][col] = sum;
  __syncthreads();
  if (at == 0) {
    for (int w = 1; w < 64; ++w) sum += part[w][col];
    a.sink_sum[((int64_t)b * a.hkv + h) * words + e] = sum;
  }
}

// Sums of dS per position over the query tiles, 16 positions of one head a
// workgroup: 64 threads a position take every 64th tile, and their sums are
// added in order.
__global__ __launch_bounds__(1024) void window_bias_sum_kernel(WinArgs a) {
  __shared__ float part[64][17];
  const int n_pos = 2 * a.range + 1, col = threadIdx.x & 15, at = threadIdx.x >> 4;
  const int head = blockIdx.x, m = blockIdx.y * 16 + col;
  float sum = 0.0f;
  if (m < n_pos)
    for (int t = at; t < a.n_tiles; t += 64)
      sum += a.bias_part[((int64_t)t * a.hq + head) * n_pos + m];
  part[at][col] = sum;
  __syncthreads();
  if (at == 0 && m < n_pos) {
    for (int w = 1; w < 64; ++w) sum += part[w][col];
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
  float *nlse, *ndelta, *sink_part, *sink_sum, *bias_part, *bias_sum, *head_part;
};

// Whether any query may have left the first tokens behind its window.
static bool has_sinks(int64_t nk, int64_t left, int64_t sinks) {
  return sinks > 0 && left >= 0 && left < nk - 1;
}

// Parts of a group's heads in the dK/dV kernel: as many as it takes to have
// about four workgroups per CU (4096 tokens, 32 / 2 heads of 32, windows of 512:
// the backward 64 us, 179 unsplit; 32768 tokens: 377 and 403, in 2 parts; with 4 kv
// heads of 64 at 32768 tokens there is one part either way).
static int head_splits(int64_t nk, int64_t hkv, int64_t g, int64_t batch) {
  const int64_t items = win_tiles(nk, WIN_KEYS, batch) * hkv;
  const int64_t splits = (1024 + items - 1) / items;
  return (int)(splits < g ? splits : g);
}

static void carve(Carver& c, WinBwdWs& w, int64_t nq, int64_t nk, int64_t hq, int64_t hkv,
                  int64_t d, int64_t batch, int64_t left, int64_t sinks, int64_t range) {
  w = WinBwdWs{};
  w.nlse = c.take<float>((size_t)(nq * hq));
  w.ndelta = c.take<float>((size_t)(nq * hq));
  if (has_sinks(nk, left, sinks)) {
    w.sink_part = c.take<float>((size_t)win_tiles(nq, WIN_SINK_QUERIES, batch) * hq * 2 * sinks *
                                d);
    w.sink_sum = c.take<float>((size_t)batch * hkv * 2 * sinks * d);
  }
  const int splits = head_splits(nk, hkv, hq / hkv, batch);
  if (splits > 1) w.head_part = c.take<float>((size_t)splits * nk * hkv * 2 * d);
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
                         dim3(win_grid((int64_t)a.n_sink_chunks * a.hq * ((a.sinks + 31) / 32))),
                         block, bias_lds, st, a);
      LSRM_CHECK_LAUNCH();
      if (a.batch > 0) {
        hipLaunchKernelGGL(window_sink_sum_kernel, dim3(a.batch * a.hkv, 2 * a.sinks * D / 16),
                           dim3(1024), 0, st, a, D);
        LSRM_CHECK_LAUNCH();
      }
    }
    hipLaunchKernelGGL((window_dkdv_kernel<DT, D, BIAS, false>),
                       dim3(win_grid((int64_t)a.n_key_tiles * a.hkv * a.head_splits)), block,
                       bias_lds, st, a);
    LSRM_CHECK_LAUNCH();
    if (a.head_splits > 1) {
      hipLaunchKernelGGL((window_dkdv_join_kernel<DT, D>),
                         dim3(ceil_div((int64_t)a.nk * a.hkv * (D / 2), 256)), block, 0, st, a);
      LSRM_CHECK_LAUNCH();
    }
  }
  if constexpr (BIAS) {
    hipLaunchKernelGGL(window_bias_sum_kernel, dim3(a.hq, ceil_div(2 * a.range + 1, 16)),
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
                                    const void* o, const void* o_low, const float* lse, int dtype,
                                    int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                    int64_t n_q, int64_t n_k, int64_t hq, int64_t hkv,
                                    int64_t head_dim, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, int64_t batch, int64_t left,
                                    int64_t right, int64_t sinks, const void* bias_table,
                                    int64_t n_buckets, const int32_t* bias_buckets,
                                    int64_t bias_range, float softmax_scale, void* dq, void* dk,
                                    void* dv, void* d_table, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  WinArgs a;
  const int rc = win_args(a, q, k, v, dtype, q_stride, k_stride, v_stride, n_q, n_k, hq, hkv,
                          head_dim, cu_seqlens_q, cu_seqlens_k, batch, left, right, sinks,
                          bias_table, n_buckets, bias_buckets, bias_range, softmax_scale);
  if (rc) return rc;
  if ((n_q > 0 && (!dout || !o || !lse || !dq)) || (n_k > 0 && (!dk || !dv)) ||
      (bias_table != nullptr) != (d_table != nullptr))
    return LSRM_ERR_INVALID_ARG;
  if (((uintptr_t)dout | (uintptr_t)o | (uintptr_t)o_low | (uintptr_t)dq | (uintptr_t)dk |
       (uintptr_t)dv) & 15u)
    return LSRM_ERR_UNSUPPORTED;
  if (hq * head_dim > WIN_MAX_STRIDE) return LSRM_ERR_UNSUPPORTED;
  Carver c{(char*)workspace, 0, workspace_bytes};
  WinBwdWs w;
  carve(c, w, n_q, n_k, hq, hkv, head_dim, batch, left, sinks, bias_table ? bias_range : -1);
  if (!workspace || !c.ok()) return LSRM_ERR_WORKSPACE;
  a.dout = (const uint16_t*)dout;
  a.o = (const uint16_t*)o;
  a.o_low = (const int8_t*)o_low;
  a.lse_in = lse;
  a.out = (uint16_t*)dq;
  a.dk = (uint16_t*)dk;
  a.dv = (uint16_t*)dv;
  a.nlse = w.nlse;
  a.ndelta = w.ndelta;
  a.head_part = w.head_part;
  a.head_splits = head_splits(n_k, hkv, hq / hkv, batch);
  a.sink_part = w.sink_part;
  a.sink_sum = w.sink_sum;
  a.bias_part = w.bias_part;
  a.bias_sum = w.bias_sum;
  a.dtable = (uint16_t*)d_table;
  a.n_key_tiles = win_tiles(n_k, WIN_KEYS, batch);
  a.n_sink_chunks = win_tiles(n_q, WIN_SINK_QUERIES, batch);
  if ((int64_t)a.n_key_tiles * hkv > INT32_MAX - NXCD ||
      (int64_t)a.n_sink_chunks * hq * 2 > INT32_MAX - NXCD || batch * hkv > INT32_MAX)
    return LSRM_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  return dtype == LSRM_BF16 ? bwd_dims<LSRM_BF16>(a, head_dim, st)
                            : bwd_dims<LSRM_F16>(a, head_dim, st);
}
