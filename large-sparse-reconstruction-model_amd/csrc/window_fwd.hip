// Sliding-window attention forward on bf16/fp16 MFMA (gfx950).
//
// For every query, an online softmax in base 2 over the keys that it sees
// (window.h), P rounded to the input type before P.V, O = acc / l and
// LSE = m + log2(l) in log2 units; a row that sees no key gives O = 0 and
// LSE = -inf.
//
// A workgroup is four waves of 32 queries of one head each; 64 keys at a time
// are copied straight to LDS, two buffers.  Scores are S^T = K Q^T, a lane's of
// one query, so the softmax exchanges nothing between lanes but the halves' sum
// at the end, and P is the operand of O^T = V^T P^T as it stands; V is read
// transposed from LDS.
//
// Bound by the issue of one SIMD: its matrix and its vector instructions take
// turns (two waves of each took the sum of both times).  32 queries by 32 keys at
// head dim 64 are 256 cycles of MFMA and some 420 of vector work (16 exponentials
// of 8 cycles, scaling, rounding, sums, and the rows' beginning and end), 680 of
// the 805 that they take.  65536 tokens, 24 heads of 64, windows of 1024: 568 us,
// 720 TFLOP/s; 2048 queries of 4 sequences behind 16384 keys each, 32 / 8 heads
// of 128, fp16, windows of 4096: 160 us, 860 TFLOP/s.  Tried without gain: two key
// blocks at once, V read ahead of the exponentials, instructions of both kinds
// interleaved by hand.
#include "window.h"

namespace lsrm {

// The softmax reference of a row is the maximum of the first block in which it
// sees a key, and follows the maximum only where a lane's sum of 16 new P
// passes this limit: P = 2^60 is as exact as P = 1 in bf16 and fp32, fp16 ends
// at 2^16.  That saves the maximum of every block, a tenth of its vector work.
template <int DT>
constexpr float WIN_LIMIT = DT == LSRM_F16 ? 4096.0f : 1152921504606846976.0f;

// One row by definition, touching the keys that it sees and no others: taken
// for rows whose output is not finite although their scores are, since a value
// that is not finite reaches the rows of its tile that mask it (0 * inf).  All
// lanes of a wave; lane = key for the scores, lane = channel for P.V.
template <int DT, int D, bool BIAS>
__device__ inline __attribute__((always_inline)) void exact_row(const WinArgs& a, const WinSeq& s,
                                                                int h, int hh, int64_t qi, int p,
                                                                const float* bias) {
  const int lane = lane_id();
  const int lo = p - a.left > 0 ? p - a.left : 0;
  int hi = p + a.right + 1;
  hi = hi < s.lk ? hi : s.lk;
  const int ns = a.sinks < lo ? a.sinks : lo, n = hi > 0 ? ns + hi - lo : 0;
  const uint16_t* q = a.q + qi * a.q_stride + (int64_t)hh * D;
  constexpr int ND = (D + 63) / 64;
  float m = -__builtin_inf(), l = 0.0f, o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i] = 0.0f;
  for (int base = 0; base < n; base += 64) {
    const int at = base + lane;
    const int j = at < ns ? at : at - ns + lo;
    float sc = -__builtin_inf();
    if (at < n) {
      const uint16_t* k = a.k + (int64_t)(s.k0 + j) * a.k_stride + (int64_t)h * D;
      float x = 0.0f;
      for (int d = 0; d < D; ++d) x = __builtin_fmaf(to_f32<DT>(q[d]), to_f32<DT>(k[d]), x);
      sc = x * a.scale_log2;
      if constexpr (BIAS) {
        int r = j - p;
        r = r < -a.range ? -a.range : (r > a.range ? a.range : r);
        sc += bias[WIN_PAD + a.range + r];
      }
    }
    float top = sc;
    for (int w = 32; w > 0; w >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, w));
    const float m_new = __builtin_elementwise_maximum(m, top);
    if (m_new == -__builtin_inf()) continue;
    const float alpha = m == -__builtin_inf() ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    const float pr = __builtin_amdgcn_exp2f(sc - m);
    float sum = pr;
    for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
    l = l * alpha + sum;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] *= alpha;
    const int cnt = n - base < 64 ? n - base : 64;
    for (int t = 0; t < cnt; ++t) {
      const float pt = __shfl(pr, t), st = __shfl(sc, t);
      if (st == -__builtin_inf()) continue;  // masked by the bias
      const int jt = base + t < ns ? base + t : base + t - ns + lo;
      const uint16_t* v = a.v + (int64_t)(s.k0 + jt) * a.v_stride + (int64_t)h * D;
#pragma unroll
      for (int i = 0; i < ND; ++i)
        if (i * 64 + lane < D) o[i] = __builtin_fmaf(pt, to_f32<DT>(v[i * 64 + lane]), o[i]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
    if (i * 64 + lane < D) {
      const int64_t at = (qi * a.hq + hh) * D + i * 64 + lane;
      const uint32_t hi = stored_bits(from_f32<DT>(o[i] * inv));
      a.out[at] = (uint16_t)hi;
      if (a.out_low)
        a.out_low[(qi * a.hq + hh) * D + low_at<D>(i * 64 + lane)] =
            (int8_t)(low_part<DT>(o[i] * inv, hi) >> LOW_SHIFT<DT>);
    }
}

template <int DT, int D, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 4))) void
window_fwd_kernel(WinArgs a) {
  using G = KvTile<D>;
  constexpr int NS = D / 16, ND = D / 32;
  __shared__ __align__(1024) char sK[2][G::BYTES];
  __shared__ __align__(1024) char sV[2][G::BYTES];
  extern __shared__ float s_bias[];

  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
  const int hb = lane >> 5, l32 = lane & 31;
  const int item = win_item();
  const int groups = a.g >> a.gt_log2;  // head groups of a kv head
  if (item >= a.n_tiles * a.hkv * groups) return;
  const int head_group = item / a.n_tiles;
  const int h = head_group / groups;
  const int tq = 128 >> a.gt_log2;  // queries per tile
  int idx;
  const WinSeq s =
      win_sequence(a, win_find(a.cu_q, a.batch, a.nq, tq, item % a.n_tiles, &idx));
  if (idx < 0 || (int64_t)idx * tq >= s.lq) return;
  const int i0 = idx * tq;
  const int qn = s.lq - i0 < tq ? s.lq - i0 : tq;
  const int lk = s.b < a.batch ? s.lk : 0;

  // This wave: 32 consecutive queries of one head.
  const int gt_mask = (1 << a.gt_log2) - 1;
  const int hh = h * a.g + ((head_group % groups) << a.gt_log2) + (wv & gt_mask);
  const int r0 = (wv >> a.gt_log2) * 32;
  const bool row_ok = r0 + l32 < qn;
  const int pos0 = i0 + lk - s.lq;  // position of the tile's first query
  const int p = pos0 + r0 + l32;
  const int64_t qi = (int64_t)s.q0 + i0 + r0 + l32;

  // Keys of the tile: the first tokens that lie before its windows (one key
  // tile), then the span of its windows, 64 keys at a time.
  const int p_last = pos0 + qn - 1;
  const int lo = pos0 - a.left > 0 ? pos0 - a.left : 0;
  int hi = p_last + a.right + 1;
  hi = hi < lk ? hi : lk;
  const int ns = hi > 0 ? (a.sinks < lo ? a.sinks : lo) : 0;
  const int st = ns > 0 ? 1 : 0;
  const int nt = st + (hi > lo ? (hi - lo + KT - 1) / KT : 0);
  // Of this wave: its first and last row (rows past the end count as the last).
  const int w_first = pos0 + r0, w_last = w_first + 31 < p_last ? w_first + 31 : p_last;
  const bool wave_on = r0 < qn;
  const int w_lo = w_first - a.left;
  int w_hi = w_last + a.right + 1;
  w_hi = w_hi < lk ? w_hi : lk;
  // Every row sees the keys from w_last - left to here.
  const int w_all = w_first + a.right + 1 < lk ? w_first + a.right + 1 : lk;
  // Of this lane's row.
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

  u32x4 qb[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i)
    qb[i] = row_ok ? *reinterpret_cast<const u32x4*>(a.q + qi * a.q_stride + (int64_t)hh * D +
                                                     i * 16 + hb * 8)
                   : u32x4{0u, 0u, 0u, 0u};
  TransposedRead<D> tr;
  tr.init(lane);

  const float* bias = nullptr;
  if constexpr (BIAS) {
    const int len = win_bias_len(a.range);
    win_load_bias<DT>(a, hh - (wv & gt_mask), gt_mask + 1, s_bias, tid);
    bias = s_bias + (wv & gt_mask) * len;
  }

  f32x16 oacc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) oacc[i][v] = 0.0f;
  float m_run = -__builtin_inf(), l_run = 0.0f;

  // One 32-key block: keys k0 .. k0 + 31, `cnt` of them in the tile.
  auto body = [&](const char* ks, const char* vs, int k0, int cnt)
      __attribute__((always_inline)) {
    f32x16 sc;
#pragma unroll
    for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
      sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(ks + G::off(l32, 2 * i + hb)), qb[i], sc);
    if constexpr (BIAS) {
      // Scores to log2 units, with the bias; one value for keys outside (-R, R).
      const int rel_lo = k0 - w_last, rel_hi = k0 + 31 - w_first;
      if (rel_hi <= -a.range || rel_lo >= a.range) {
        const float c = bias[WIN_PAD + (rel_lo >= a.range ? 2 * a.range : 0)];
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = __builtin_fmaf(sc[v], a.scale_log2, c);
      } else {
        const float* at = bias + WIN_PAD + a.range + k0 - p + hb * 4;
#pragma unroll
        for (int v = 0; v < 16; ++v)
          sc[v] = __builtin_fmaf(sc[v], a.scale_log2, at[acc_row(v, 0)]);
      }
    }
    if (k0 + 32 > w_all || k0 < w_last - a.left || cnt < 32) {
      const int end = k0 + cnt < row_hi ? k0 + cnt : row_hi, base = k0 + hb * 4;
      const uint32_t seen = bits_below(end - base) &
                            (~bits_below(row_lo - base) | bits_below(a.sinks - base));
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = keep(seen, v, sc[v], -__builtin_inf());
    }
    // The rows' references follow the block's maxima.
    auto follow = [&]() __attribute__((always_inline)) {
      asm volatile("");  // (a branch, not both sides and a selection)
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = sc[i];
      float m_new = half_max(max_of<16>(x));
      if constexpr (!BIAS) m_new *= a.scale_log2;
      m_new = __builtin_elementwise_maximum(m_run, m_new);
      const float alpha =
          m_new == -__builtin_inf() ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) oacc[i][v] *= alpha;
    };
    u32x4 pb[2];
    auto probabilities = [&]() __attribute__((always_inline)) {
      const float negm = m_run == -__builtin_inf() ? 0.0f : -m_run;
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v0 = c * 8 + 2 * e;
          float x0, x1;
          if constexpr (BIAS) {
            x0 = sc[v0] + negm;
            x1 = sc[v0 + 1] + negm;
          } else {
            x0 = __builtin_fmaf(sc[v0], a.scale_log2, negm);
            x1 = __builtin_fmaf(sc[v0 + 1], a.scale_log2, negm);
          }
          pb[c][e] = pack2<DT>(__builtin_amdgcn_exp2f(x0), __builtin_amdgcn_exp2f(x1));
          sum = sum2<DT>(pb[c][e], sum);
        }
      return sum;
    };
    const bool fresh = __builtin_amdgcn_ballot_w64(m_run == -__builtin_inf()) != 0;
    if (fresh) follow();
    float sum = probabilities();
    if (__builtin_amdgcn_ballot_w64(!(sum <= WIN_LIMIT<DT>)) != 0 && !fresh) {
      follow();
      sum = probabilities();
    }
    l_run += sum;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < ND; ++db)
        oacc[db] = mfma32<DT>(tr.read(vs, db, c * 16), pb[c], oacc[db]);
  };

  for (int t = 0; t < nt; ++t) {
    wait_copies();
    __syncthreads();
    if (t + 1 < nt) load(t + 1);
    int a0, cnt;
    tile_at(t, &a0, &cnt);
    if (!wave_on) continue;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int k0 = a0 + blk * 32, left = cnt - blk * 32;
      if (left > 0 && k0 < w_hi && (k0 + 32 > w_lo || k0 < a.sinks))
        body(sK[t & 1] + blk * 32 * (D * 2), sV[t & 1] + blk * 32 * (D * 2), k0, left);
    }
  }

  if (!wave_on) return;
  const float l_tot = half_sum(l_run);
  const float inv = l_tot > 0.0f ? 1.0f / l_tot : (l_tot == 0.0f ? 0.0f : l_tot);
  bool odd = false;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      if (l_tot == 0.0f) oacc[db][v] = 0.0f;
      odd |= !(__builtin_fabsf(oacc[db][v]) < __builtin_inf());
    }
  // The halves of a wave hold four of every eight columns each; swapped, a lane
  // has eight columns of every sixteen, in 16-byte stores.
  uint32_t low[ND * 4];
  uint16_t* orow = a.out + (qi * a.hq + hh) * D + hb * 8;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = oacc[i / 2][(i % 2) * 8 + e] * inv;
    uint32_t w0 = stored_bits(pack2<DT>(x[0], x[1]));
    uint32_t w1 = stored_bits(pack2<DT>(x[2], x[3]));
    uint32_t w2 = stored_bits(pack2<DT>(x[4], x[5]));
    uint32_t w3 = stored_bits(pack2<DT>(x[6], x[7]));
    if (a.out_low) {
      low[i * 2] = low_word<DT>(x, w0, w1);
      low[i * 2 + 1] = low_word<DT>(x + 4, w2, w3);
      swap_halves(low[i * 2], low[i * 2 + 1]);
    }
    swap_halves(w0, w2);
    swap_halves(w1, w3);
    if (row_ok) *reinterpret_cast<u32x4*>(orow + i * 16) = u32x4{w0, w1, w2, w3};
  }
  if (row_ok) {
    if (a.out_low) {
      u32x4* at = reinterpret_cast<u32x4*>(a.out_low + (qi * a.hq + hh) * D + hb * (D / 2));
#pragma unroll
      for (int i = 0; i < ND; ++i)
        at[i] = u32x4{low[i * 4], low[i * 4 + 1], low[i * 4 + 2], low[i * 4 + 3]};
    }
    if (hb == 0 && a.lse)
      a.lse[(int64_t)hh * a.nq + qi] =
          l_tot == 0.0f ? -__builtin_inf() : m_run + log2f(l_tot);
  }
  // Finite sums over scores, but a value that is not finite in the output.
  uint64_t redo = __builtin_amdgcn_ballot_w64(row_ok && odd && l_tot > 0.0f &&
                                              l_tot < __builtin_inf());
  redo = (redo | (redo >> 32)) & 0xffffffffull;
  while (redo) {
    const int r = __builtin_ctzll(redo);
    redo &= redo - 1;
    exact_row<DT, D, BIAS>(a, WinSeq{s.b, s.q0, s.lq, s.k0, lk}, h, hh,
                           (int64_t)s.q0 + i0 + r0 + r, pos0 + r0 + r, bias);
  }
}

template <int DT, int D>
static int fwd_launch(const WinArgs& a, hipStream_t st) {
  const int grid = win_grid((int64_t)a.n_tiles * a.hkv * (a.g >> a.gt_log2));
  if (a.table) {
    const size_t lds = (size_t)(win_bias_len(a.range) << a.gt_log2) * 4;
    hipLaunchKernelGGL((window_fwd_kernel<DT, D, true>), dim3(grid), dim3(256), lds, st, a);
  } else {
    hipLaunchKernelGGL((window_fwd_kernel<DT, D, false>), dim3(grid), dim3(256), 0, st, a);
  }
  LSRM_CHECK_LAUNCH();
  return LSRM_OK;
}

// Checks shared by the forward and backward entry points; fills the launch
// arguments that both use.
int win_args(WinArgs& a, const void* q, const void* k, const void* v, int dtype, int64_t q_stride,
             int64_t k_stride, int64_t v_stride, int64_t nq, int64_t nk, int64_t hq, int64_t hkv,
             int64_t d, const int32_t* cu_q, const int32_t* cu_k, int64_t batch, int64_t left,
             int64_t right, int64_t sinks, const void* table, int64_t n_buckets,
             const int32_t* buckets, int64_t range, float scale) {
  if (dtype != LSRM_BF16 && dtype != LSRM_F16) return LSRM_ERR_UNSUPPORTED;
  if (d != 32 && d != 64 && d != 128) return LSRM_ERR_UNSUPPORTED;
  if (nq < 0 || nk < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || batch < 0 || left < -1 ||
      right < -1 || sinks < 0)
    return LSRM_ERR_INVALID_ARG;
  if (!(scale > 0.0f) || !(scale < __builtin_inff())) return LSRM_ERR_INVALID_ARG;
  if ((table != nullptr) != (buckets != nullptr) ||
      (table && (n_buckets <= 0 || range < 0)))
    return LSRM_ERR_INVALID_ARG;
  if (nq > WIN_MAX_TOKENS || nk > WIN_MAX_TOKENS || batch > WIN_MAX_TOKENS || hq > 65535 ||
      sinks > WIN_MAX_SINKS || (table && (range > WIN_MAX_RANGE || n_buckets > (1 << 20))))
    return LSRM_ERR_UNSUPPORTED;
  // rows are read in 16-byte pieces
  if (q_stride < hq * d || k_stride < hkv * d || v_stride < hkv * d) return LSRM_ERR_INVALID_ARG;
  if (q_stride % 8 || k_stride % 8 || v_stride % 8 || q_stride > WIN_MAX_STRIDE ||
      k_stride > WIN_MAX_STRIDE || v_stride > WIN_MAX_STRIDE)
    return LSRM_ERR_UNSUPPORTED;
  if (nq > 0 && (!q || !cu_q || !cu_k)) return LSRM_ERR_INVALID_ARG;
  if (nk > 0 && (!k || !v || !cu_q || !cu_k)) return LSRM_ERR_INVALID_ARG;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15u) return LSRM_ERR_UNSUPPORTED;
  a = WinArgs{};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.nq = (int)nq;
  a.nk = (int)nk;
  a.batch = (int)batch;
  a.hq = (int)hq;
  a.hkv = (int)hkv;
  a.g = (int)(hq / hkv);
  // The waves of a workgroup share the tiles of one kv head: as many of its query
  // heads as divide the group (32768 tokens, windows of 512, forward and backward:
  // 32 / 2 heads of 32 147 and 377 us, one head a workgroup 162 and 388; 1024
  // tokens 11.9 and 16.2, 36 and 41), the rest of the waves more queries.
  a.gt_log2 = a.g % 4 == 0 ? 2 : (a.g % 2 == 0 ? 1 : 0);
  a.n_tiles = win_tiles(nq, 128 >> a.gt_log2, batch);
  // -1 (no bound) and anything longer than a sequence
  a.left = (int)(left < 0 || left > WIN_MAX_TOKENS ? WIN_MAX_TOKENS : left);
  a.right = (int)(right < 0 || right > WIN_MAX_TOKENS ? WIN_MAX_TOKENS - 1 : right);
  a.sinks = (int)sinks;
  a.scale = scale;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.table = (const uint16_t*)table;
  a.buckets = buckets;
  a.n_buckets = (int)n_buckets;
  a.range = table ? (int)range : 0;
  if ((int64_t)a.n_tiles * hq > INT32_MAX - NXCD) return LSRM_ERR_UNSUPPORTED;
  return LSRM_OK;
}

}  // namespace lsrm

using namespace lsrm;

namespace lsrm {
// One workgroup: the flag word of lsrm_window_validate.
__global__ __launch_bounds__(256) void window_validate_kernel(
    const int32_t* cu_q, const int32_t* cu_k, int batch, int nq, int nk, const int32_t* buckets,
    int n_pos, int n_buckets, int32_t* flags) {
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i <= batch; i += 256) {
    const int q = cu_q[i], k = cu_k[i];
    const int q1 = i < batch ? cu_q[i + 1] : nq, k1 = i < batch ? cu_k[i + 1] : nk;
    if (q > q1 || k > k1 || q < 0 || k < 0 || (i == 0 && (q != 0 || k != 0)))
      mine |= LSRM_META_SEQLENS_BAD;
  }
  for (int i = threadIdx.x; i < n_pos; i += 256)
    if (buckets[i] < 0 || buckets[i] >= n_buckets) mine |= LSRM_META_BUCKETS_BAD;
  if (mine) atomicOr(&bad, mine);
  __syncthreads();
  // seen by the host as soon as it is written, where the word is in its memory
  if (threadIdx.x == 0)
    __hip_atomic_store(flags, bad, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}
}  // namespace lsrm

extern "C" int lsrm_window_validate(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                    int64_t batch, int64_t n_q, int64_t n_k,
                                    const int32_t* bias_buckets, int64_t bias_range,
                                    int64_t n_buckets, int32_t* flags, void* stream) {
  if (!cu_seqlens_q || !cu_seqlens_k || !flags || batch < 0 || n_q < 0 || n_k < 0 ||
      (bias_buckets && (bias_range < 0 || n_buckets <= 0)))
    return LSRM_ERR_INVALID_ARG;
  if (n_q > WIN_MAX_TOKENS || n_k > WIN_MAX_TOKENS || batch > WIN_MAX_TOKENS ||
      (bias_buckets && (bias_range > WIN_MAX_RANGE || n_buckets > (1 << 20))))
    return LSRM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(window_validate_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream,
                     cu_seqlens_q, cu_seqlens_k, (int)batch, (int)n_q, (int)n_k, bias_buckets,
                     bias_buckets ? (int)(2 * bias_range + 1) : 0, (int)n_buckets, flags);
  LSRM_CHECK_LAUNCH();
  return LSRM_OK;
}

extern "C" int lsrm_window_attn_fwd(const void* q, const void* k, const void* v, int dtype,
                                    int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                    int64_t n_q, int64_t n_k, int64_t hq, int64_t hkv,
                                    int64_t head_dim, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, int64_t batch, int64_t left,
                                    int64_t right, int64_t sinks, const void* bias_table,
                                    int64_t n_buckets, const int32_t* bias_buckets,
                                    int64_t bias_range, float softmax_scale, void* out,
                                    void* out_low, float* lse, void* stream) {
  WinArgs a;
  const int rc = win_args(a, q, k, v, dtype, q_stride, k_stride, v_stride, n_q, n_k, hq, hkv,
                          head_dim, cu_seqlens_q, cu_seqlens_k, batch, left, right, sinks,
                          bias_table, n_buckets, bias_buckets, bias_range, softmax_scale);
  if (rc) return rc;
  if (n_q == 0) return LSRM_OK;
  if (!out) return LSRM_ERR_INVALID_ARG;
  if (((uintptr_t)out | (uintptr_t)out_low) & 15u) return LSRM_ERR_UNSUPPORTED;
  a.out = (uint16_t*)out;
  a.out_low = (int8_t*)out_low;
  a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSRM_BF16) {
    if (head_dim == 32) return fwd_launch<LSRM_BF16, 32>(a, st);
    if (head_dim == 64) return fwd_launch<LSRM_BF16, 64>(a, st);
    return fwd_launch<LSRM_BF16, 128>(a, st);
  }
  if (head_dim == 32) return fwd_launch<LSRM_F16, 32>(a, st);
  if (head_dim == 64) return fwd_launch<LSRM_F16, 64>(a, st);
  return fwd_launch<LSRM_F16, 128>(a, st);
}
