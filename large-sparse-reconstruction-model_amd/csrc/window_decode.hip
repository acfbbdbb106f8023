// Sliding-window attention of single query tokens against a cache (gfx950).
//
// The query of a sequence of n cached tokens stands at position n - 1 and sees
// keys n - 1 - left .. n - 1 and the first `sinks` tokens.  All of them are
// read once and nothing else is: the kernel is bound by those bytes, or by
// latency where there are few.  The query heads of a kv head (32 at most per
// workgroup) share one read of its keys and values.
//
// A workgroup takes one kv head of one sequence and one of `splits` parts of
// its keys; its four waves take 32-key blocks in turn, each at its own pace:
// a wave copies a block's K and V rows straight to its own LDS, the next block
// in flight, and waits for its own copies only.  Scores are S^T = K Q^T, one
// head per lane, O^T = V^T P^T; the waves' sums are joined in LDS and the
// parts' by a second launch, in a fixed order, in fp32.
//
// 256 sequences of up to 4096 tokens, 24 heads of 64, windows of 2048: 510 us, 6.2
// TB/s (a copy of 2 GiB moves 4.9, reads and writes); 64 sequences, 16 / 4 heads
// of 128, windows of 1024: 25 us, 4.8 TB/s; one sequence of 4096 keys, 32 / 2 heads
// of 64: 7.6 us, two launches.
#include "window.h"

namespace lsrm {

struct DecodeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_batch, k_token, k_head, v_batch, v_token, v_head;
  const int32_t* lens;
  int batch, capacity, hq, hkv, g, chunks, splits;  // chunks: of 32 heads of a group
  int items, left, sinks;
  float scale_log2;
  WinArgs bias;        // table, buckets, n_buckets, range, hq
  uint16_t* out;
  float* lse;          // [hq, batch] log2 units, or null
  float* part;         // [batch, hq, splits, d + 2]: O, maximum, sum
};

// Wait until at most N of this wave's vector-memory loads are in flight.
template <int N>
__device__ inline void wait_loads() {
  static_assert(N < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

template <int DT, int D, bool BIAS>
__global__ __launch_bounds__(256) void window_decode_kernel(DecodeArgs a) {
  using G = KvTile<D>;
  constexpr int NS = D / 16, ND = D / 32, KPL = G::KPL, LOADS = 32 / KPL, BYTES = 32 * D * 2;
  constexpr int RED = ND * 16 + 2;  // words per lane of a wave's sums
  static_assert(3 * RED * 64 * 4 <= 4 * 4 * BYTES, "the waves' sums fit where their blocks were");
  __shared__ __align__(1024) char s_kv[4][2][2][BYTES];  // wave, buffer, K / V
  const int lane = lane_id(), wv = uniform(wave_id());
  const int hb = lane >> 5, l32 = lane & 31;
  int item = win_item();  // neighbouring heads share cache lines where D = 32
  if (item >= a.items) return;
  const int split = item % a.splits;
  item /= a.splits;
  const int chunk = item % a.chunks;
  item /= a.chunks;
  const int h = item % a.hkv, b = item / a.hkv;
  int n = a.lens[b];
  n = n < 0 ? 0 : (n > a.capacity ? a.capacity : n);
  const int lo = n - 1 - a.left > 0 ? n - 1 - a.left : 0;
  const int ns = a.sinks < lo ? a.sinks : lo;
  // Blocks of 32 keys: the first tokens before the window, then the window.
  const int sink_blocks = (ns + 31) / 32, blocks = sink_blocks + (n - lo + 31) / 32;
  const int per = (blocks + a.splits - 1) / a.splits;
  const int first = split * per, last = first + per < blocks ? first + per : blocks;

  const int heads = a.g - chunk * 32 < 32 ? a.g - chunk * 32 : 32;
  const bool head_ok = l32 < heads;
  const int hh = h * a.g + chunk * 32 + (head_ok ? l32 : 0);
  u32x4 qb[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i)
    qb[i] = head_ok ? *reinterpret_cast<const u32x4*>(a.q + (int64_t)b * a.q_stride +
                                                      (int64_t)hh * D + i * 16 + hb * 8)
                    : u32x4{0u, 0u, 0u, 0u};
  TransposedRead<D> tr;
  tr.init(lane);

  const uint16_t* kh = a.k + (int64_t)b * a.k_batch + (int64_t)h * a.k_head;
  const uint16_t* vh = a.v + (int64_t)b * a.v_batch + (int64_t)h * a.v_head;
  auto block_at = [&](int t, int* a0, int* cnt) __attribute__((always_inline)) {
    const int end = t < sink_blocks ? ns : n;
    *a0 = t < sink_blocks ? t * 32 : lo + (t - sink_blocks) * 32;
    *cnt = end - *a0 < 32 ? end - *a0 : 32;
  };
  auto copy = [&](const uint16_t* base, uint32_t row_bytes, int cnt, char* dst)
      __attribute__((always_inline)) {
    const uint32_t d0 = (uint32_t)uniform((int)lds_addr(dst));
    base = uniform_ptr(base);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int row = j * KPL + lane / G::CH, from = row < cnt ? row : cnt - 1;
      copy16_to_lds(base,
                    (uint32_t)from * row_bytes + (((lane % G::CH) ^ G::swz(row)) << 4),
                    d0 + j * 1024);
    }
  };
  auto load = [&](int t, int buf) __attribute__((always_inline)) {
    int a0, cnt;
    block_at(t, &a0, &cnt);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the buffer's reads have returned
    copy(kh + (int64_t)a0 * a.k_token, (uint32_t)a.k_token * 2, cnt, s_kv[wv][buf][0]);
    copy(vh + (int64_t)a0 * a.v_token, (uint32_t)a.v_token * 2, cnt, s_kv[wv][buf][1]);
  };

  f32x16 oacc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) oacc[i][v] = 0.0f;
  float m_run = -__builtin_inf(), l_run = 0.0f;
  float far = 0.0f;
  if constexpr (BIAS) far = win_bias_at<DT>(a.bias, hh, 0);

  const int t0 = first + wv;
  wait_loads<0>();  // the query: from here on only copies are in flight
  if (t0 < last) load(t0, 0);
  int buf = 0;
  for (int t = t0; t < last; t += 4, buf ^= 1) {
    if (t + 4 < last) {
      load(t + 4, buf ^ 1);
      wait_loads<2 * LOADS>();
    } else {
      wait_loads<0>();
    }
    wave_lds_order();
    int a0, cnt;
    block_at(t, &a0, &cnt);
    const char* ks = s_kv[wv][buf][0];
    const char* vs = s_kv[wv][buf][1];
    f32x16 sc;
#pragma unroll
    for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
      sc = mfma32<DT>(*reinterpret_cast<const u32x4*>(ks + G::off(l32, 2 * i + hb)), qb[i], sc);
    if constexpr (BIAS) {
      const int r = a.bias.range, rel = a0 - (n - 1);  // of the block's first key
      if (rel + 31 <= -r) {
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = __builtin_fmaf(sc[v], a.scale_log2, far);
      } else {
        // at most R / 32 + 1 blocks of a sequence
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          int m = rel + acc_row(v, hb) + r;
          m = m < 0 ? 0 : (m > r ? r : m);  // keys past the query are masked below
          sc[v] = __builtin_fmaf(sc[v], a.scale_log2, win_bias_at<DT>(a.bias, hh, m));
        }
        wait_loads<0>();
      }
    }
    if (cnt < 32) {
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (acc_row(v, hb) >= cnt) sc[v] = -__builtin_inf();
    }
    float top = sc[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) top = __builtin_elementwise_maximum(top, sc[v]);
    top = half_max(top);
    if constexpr (!BIAS) top *= a.scale_log2;
    if (__builtin_amdgcn_ballot_w64(!(top <= m_run)) != 0) {
      const float m_new = __builtin_elementwise_maximum(m_run, top);
      const float alpha = m_new == -__builtin_inf() ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) oacc[i][v] *= alpha;
    }
    const float negm = m_run == -__builtin_inf() ? 0.0f : -m_run;
    u32x4 pb[2];
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
        l_run = sum2<DT>(pb[c][e], l_run);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < ND; ++db)
        oacc[db] = mfma32<DT>(tr.read(vs, db, c * 16), pb[c], oacc[db]);
    wave_lds_order();
  }

  // The waves' sums, in wave order.
  l_run = half_sum(l_run);
  __syncthreads();
  float* red = reinterpret_cast<float*>(&s_kv[0][0][0][0]) + lane;
  if (wv > 0) {
    float* mine = red + (wv - 1) * RED * 64;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) mine[(db * 16 + v) * 64] = oacc[db][v];
    mine[ND * 16 * 64] = m_run;
    mine[(ND * 16 + 1) * 64] = l_run;
  }
  __syncthreads();
  if (wv > 0) return;
  float m = m_run;
#pragma unroll
  for (int w = 0; w < 3; ++w)
    m = __builtin_elementwise_maximum(m, red[(w * RED + ND * 16) * 64]);
  auto weight = [&](float mw) {
    return mw == -__builtin_inf() ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
  };
  const float f0 = weight(m_run);
  l_run *= f0;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) oacc[db][v] *= f0;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    const float* o = red + w * RED * 64;
    const float f = weight(o[ND * 16 * 64]);
    l_run = __builtin_fmaf(f, o[(ND * 16 + 1) * 64], l_run);
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        oacc[db][v] = __builtin_fmaf(f, o[(db * 16 + v) * 64], oacc[db][v]);
  }
  if (!head_ok) return;
  if (a.splits > 1) {
    float* p = a.part + (((int64_t)b * a.hq + hh) * a.splits + split) * (D + 2);
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) p[db * 32 + acc_row(v, hb)] = oacc[db][v];
    if (hb == 0) {
      p[D] = m;
      p[D + 1] = l_run;
    }
    return;
  }
  const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
  uint16_t* orow = a.out + ((int64_t)b * a.hq + hh) * D;
#pragma unroll
  for (int db = 0; db < ND; ++db)
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
      const int v = gi * 4;
      *reinterpret_cast<u32x2*>(orow + db * 32 + gi * 8 + hb * 4) =
          u32x2{pack2<DT>(oacc[db][v] * inv, oacc[db][v + 1] * inv),
                pack2<DT>(oacc[db][v + 2] * inv, oacc[db][v + 3] * inv)};
    }
  if (hb == 0 && a.lse)
    a.lse[(int64_t)hh * a.batch + b] = l_run == 0.0f ? -__builtin_inf() : m + log2f(l_run);
}

// One workgroup per (sequence, query head): each wave takes every fourth eight of
// the parts in order, then the waves' sums are added in order.
template <int DT, int D>
__global__ __launch_bounds__(256) void window_join_kernel(DecodeArgs a) {
  constexpr int N = (D + 63) / 64, AT_ONCE = 8;
  __shared__ float s_o[4][N * 64], s_l[4];
  const int lane = lane_id(), wv = wave_id();
  const int64_t row = blockIdx.x;
  const float* p = a.part + row * a.splits * (D + 2);
  float m = -__builtin_inf();
  for (int s = lane; s < a.splits; s += 64)
    m = __builtin_elementwise_maximum(m, p[(int64_t)s * (D + 2) + D]);
  for (int w = 32; w > 0; w >>= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, w));
  float o[N], l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int s0 = wv * AT_ONCE; s0 < a.splits; s0 += 4 * AT_ONCE) {
    float top[AT_ONCE], sum[AT_ONCE], x[AT_ONCE][N];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const float* at = p + (int64_t)(s0 + u < a.splits ? s0 + u : a.splits - 1) * (D + 2);
      top[u] = s0 + u < a.splits ? at[D] : -__builtin_inf();
      sum[u] = at[D + 1];
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] = i * 64 + lane < D ? at[i * 64 + lane] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (top[u] == -__builtin_inf()) continue;  // a part without keys
      const float f = __builtin_amdgcn_exp2f(top[u] - m);
      l = __builtin_fmaf(f, sum[u], l);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = __builtin_fmaf(f, x[u][i], o[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s_o[wv][i * 64 + lane] = o[i];
  if (lane == 0) s_l[wv] = l;
  __syncthreads();
  if (wv > 0) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    l += s_l[w];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] += s_o[w][i * 64 + lane];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * 64 + lane < D) a.out[row * D + i * 64 + lane] = from_f32<DT>(o[i] * inv);
  if (lane == 0 && a.lse)
    a.lse[(row % a.hq) * a.batch + row / a.hq] =
        l == 0.0f ? -__builtin_inf() : m + log2f(l);
}

// Parts of a sequence's keys: no more workgroups than the card holds at once
// (LDS: one per CU at head dim 128, two at 64, four at 32), and few where joining
// them costs more than they save.  32 query and 2 kv heads of 64, one sequence of
// bf16 keys: 512 keys 6.5 us whole and 7.3 in 4 parts, 4096 keys 25.7 whole, 8.2
// in 16 and 7.6 in 32 parts, 16384 keys 9.8, 9.1 and 10.0 in 32, 64 and 128 parts,
// 65536 keys 12.9 and 15.9 in 128 and 256 parts (336 whole).
static int decode_splits(int64_t batch, int64_t hkv, int64_t g, int64_t d, int64_t capacity,
                         int64_t left, int64_t sinks) {
  const int64_t items = batch * hkv * ((g + 31) / 32);
  const int64_t window = left < 0 || left + 1 > capacity ? capacity : left + 1;
  const int64_t blocks = (window + 31) / 32 + (sinks + 31) / 32;
  if (items == 0 || blocks < 20) return 1;
  int64_t splits = blocks / 8 < 128 ? blocks / 8 : 128;
  if (splits < 32) splits = blocks / 4 < 32 ? blocks / 4 : 32;
  const int64_t room = (256 * 128 / d + items - 1) / items;
  return (int)(splits < room ? splits : room);
}

template <int DT, int D>
static int decode_launch(const DecodeArgs& a, hipStream_t st) {
  const dim3 grid(win_grid(a.items)), block(256);
  if (a.bias.table)
    hipLaunchKernelGGL((window_decode_kernel<DT, D, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((window_decode_kernel<DT, D, false>), grid, block, 0, st, a);
  LSRM_CHECK_LAUNCH();
  if (a.splits > 1) {
    hipLaunchKernelGGL((window_join_kernel<DT, D>),
                       dim3((unsigned)(a.batch * a.hq)), block, 0, st, a);
    LSRM_CHECK_LAUNCH();
  }
  return LSRM_OK;
}

}  // namespace lsrm

using namespace lsrm;

extern "C" size_t lsrm_window_decode_workspace_size(int64_t batch, int64_t capacity, int64_t hq,
                                                    int64_t hkv, int64_t head_dim, int64_t left,
                                                    int64_t sinks) {
  if (batch <= 0 || capacity < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || head_dim <= 0 ||
      sinks < 0)
    return 0;
  const int splits = decode_splits(batch, hkv, hq / hkv, head_dim, capacity, left, sinks);
  return splits > 1 ? (size_t)batch * hq * splits * (head_dim + 2) * sizeof(float) + 256 : 0;
}

extern "C" int lsrm_window_decode(const void* q, const void* k, const void* v, int dtype,
                                  int64_t q_stride, int64_t k_batch_stride,
                                  int64_t k_token_stride, int64_t k_head_stride,
                                  int64_t v_batch_stride, int64_t v_token_stride,
                                  int64_t v_head_stride, const int32_t* seqlens, int64_t batch,
                                  int64_t capacity, int64_t hq, int64_t hkv, int64_t head_dim,
                                  int64_t left, int64_t sinks, const void* bias_table,
                                  int64_t n_buckets, const int32_t* bias_buckets,
                                  int64_t bias_range, float softmax_scale, void* out, float* lse,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != LSRM_BF16 && dtype != LSRM_F16) return LSRM_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return LSRM_ERR_UNSUPPORTED;
  if (batch < 0 || capacity < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || left < -1 || sinks < 0)
    return LSRM_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.0f) || !(softmax_scale < __builtin_inff())) return LSRM_ERR_INVALID_ARG;
  if ((bias_table != nullptr) != (bias_buckets != nullptr) ||
      (bias_table && (n_buckets <= 0 || bias_range < 0)))
    return LSRM_ERR_INVALID_ARG;
  if (capacity > WIN_MAX_TOKENS || batch > (1 << 20) || hq > 65535 || sinks > WIN_MAX_SINKS ||
      (bias_table && (bias_range > WIN_MAX_RANGE || n_buckets > (1 << 20))))
    return LSRM_ERR_UNSUPPORTED;
  const int64_t strides[7] = {q_stride,       k_batch_stride, k_token_stride, k_head_stride,
                              v_batch_stride, v_token_stride, v_head_stride};
  for (int64_t s : strides) {
    if (s < 0) return LSRM_ERR_INVALID_ARG;
    if (s % 8) return LSRM_ERR_UNSUPPORTED;
  }
  if (k_token_stride > WIN_MAX_STRIDE || v_token_stride > WIN_MAX_STRIDE)
    return LSRM_ERR_UNSUPPORTED;
  if (batch == 0) return LSRM_OK;
  if (!q || !seqlens || !out || (capacity > 0 && (!k || !v))) return LSRM_ERR_INVALID_ARG;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15u)
    return LSRM_ERR_UNSUPPORTED;
  DecodeArgs a{};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_stride = q_stride;
  a.k_batch = k_batch_stride;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_batch = v_batch_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.lens = seqlens;
  a.batch = (int)batch;
  a.capacity = (int)capacity;
  a.hq = (int)hq;
  a.hkv = (int)hkv;
  a.g = (int)(hq / hkv);
  a.chunks = (a.g + 31) / 32;
  a.splits = decode_splits(batch, hkv, a.g, head_dim, capacity, left, sinks);
  a.left = (int)(left < 0 || left > WIN_MAX_TOKENS ? WIN_MAX_TOKENS : left);
  a.sinks = (int)sinks;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.bias.table = (const uint16_t*)bias_table;
  a.bias.buckets = bias_buckets;
  a.bias.n_buckets = (int)n_buckets;
  a.bias.range = bias_table ? (int)bias_range : 0;
  a.bias.hq = (int)hq;
  a.out = (uint16_t*)out;
  a.lse = lse;
  if (batch * hkv * a.chunks * a.splits > INT32_MAX - NXCD) return LSRM_ERR_UNSUPPORTED;
  a.items = (int)(batch * hkv * a.chunks * a.splits);
  if (a.splits > 1) {
    Carver c{(char*)workspace, 0, workspace_bytes};
    a.part = c.take<float>((size_t)batch * hq * a.splits * (head_dim + 2));
    if (!workspace || !c.ok()) return LSRM_ERR_WORKSPACE;
  }
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSRM_BF16) {
    if (head_dim == 32) return decode_launch<LSRM_BF16, 32>(a, st);
    if (head_dim == 64) return decode_launch<LSRM_BF16, 64>(a, st);
    return decode_launch<LSRM_BF16, 128>(a, st);
  }
  if (head_dim == 32) return decode_launch<LSRM_F16, 32>(a, st);
  if (head_dim == 64) return decode_launch<LSRM_F16, 64>(a, st);
  return decode_launch<LSRM_F16, 128>(a, st);
}
