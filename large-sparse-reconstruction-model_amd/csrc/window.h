// Pieces shared by the sliding-window attention kernels (forward, backward,
// single tokens).
//
// Query i of a sequence of Lq queries and Lk keys stands at position
// p = i + Lk - Lq (the last query at the last key).  It sees key j, 0 <= j <
// Lk, where j <= p + right and (j >= p - left or j < sinks): a window, and the
// sequence's first `sinks` tokens.  A learned bias table[bucket[clamp(j - p,
// -R, R) + R]][head] may be added to its scores.
#pragma once

#include "attn.h"

namespace lsrm {

constexpr int WIN_MAX_SINKS = 64;     // one key tile
constexpr int WIN_MAX_RANGE = 512;    // R: relative positions with a bias of their own
constexpr int WIN_KEYS = 128;         // keys per workgroup of the dK/dV kernel
constexpr int WIN_SINK_QUERIES = 512; // queries per partial sum of the first tokens' dK/dV
constexpr int64_t WIN_MAX_TOKENS = int64_t{1} << 29;   // positions plus windows fit 32 bits
constexpr int64_t WIN_MAX_STRIDE = int64_t{1} << 22;   // a tile's rows span less than 2^31 bytes
// A score this low means "masked": table entries below it (the lowest values
// of bf16 and fp32) count as -inf, so that a row that sees nothing else is an
// empty row in the forward and the backward alike.
constexpr float WIN_MASKED = -1e30f;

struct WinArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  const int32_t* cu_q;
  const int32_t* cu_k;
  int nq, nk, batch;
  int hq, hkv, g;
  int gt_log2;         // log2 of the query heads that a workgroup takes together
  int n_tiles;         // query tiles (an upper bound for any offsets)
  int left, right, sinks;
  float scale, scale_log2;
  const uint16_t* table;     // [n_buckets, hq] or null
  const int32_t* buckets;    // [2 range + 1]
  int n_buckets, range;
  uint16_t* out;       // forward: O; backward: dQ
  int8_t* out_low;     // forward: what rounding took from O, or null (see low_part)
  float* lse;          // forward, or null
  // backward
  const uint16_t* o;
  const int8_t* o_low;  // or null
  const uint16_t* dout;
  const float* lse_in;
  float* nlse;         // [hq, nq]: -lse, -inf for empty rows
  float* ndelta;       // [hq, nq]: -rowsum(dO * O)
  uint16_t* dk;
  uint16_t* dv;
  float* sink_part;    // [chunk, hq, 2, sinks, d] partial sums of the first tokens
  float* sink_sum;     // [batch, hkv, 2, sinks, d]
  float* head_part;    // [head_splits, nk, hkv, 2, d] sums of a part of the heads
  int head_splits;
  float* bias_part;    // [tile, hq, 2 range + 1] partial sums of dS per position
  float* bias_sum;     // [hq, 2 range + 1]
  uint16_t* dtable;    // [n_buckets, hq]
  int n_key_tiles, n_sink_chunks;
};

// One sequence: its first query and key row and their numbers.
struct WinSeq {
  int b, q0, lq, k0, lk;
};

// Offsets as used: from 0, and within 0 .. n whatever the array holds.
__device__ inline int win_offset(const int32_t* cu, int i, int n) {
  const int x = i == 0 ? 0 : cu[i];
  return x < 0 ? 0 : (x > n ? n : x);
}

__device__ inline WinSeq win_sequence(const WinArgs& a, int b) {
  WinSeq s;
  s.b = b;
  s.q0 = win_offset(a.cu_q, b, a.nq);
  s.k0 = win_offset(a.cu_k, b, a.nk);
  if (b >= a.batch) {  // rows behind the last sequence
    s.lq = a.nq - s.q0;
    s.lk = a.nk - s.k0;
  } else {
    s.lq = win_offset(a.cu_q, b + 1, a.nq) - s.q0;
    s.lk = win_offset(a.cu_k, b + 1, a.nk) - s.k0;
  }
  if (s.lq < 0) s.lq = 0;
  if (s.lk < 0) s.lk = 0;
  return s;
}

// Sequence and tile-in-sequence of tile t, for tiles of `size` rows numbered
// so that sequence b begins at cu[b] / size + b: an upper bound of the tiles
// before it that needs no prefix sum (at most one tile of each sequence stays
// empty).  "Sequence" `batch` holds the rows behind the last one.
__device__ inline int win_find(const int32_t* cu, int batch, int n, int size, int t, int* idx) {
  int lo = 0, hi = batch;
  while (lo < hi) {  // largest b with cu[b] / size + b <= t
    const int mid = (lo + hi + 1) >> 1;
    if (win_offset(cu, mid, n) / size + mid <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  lo = uniform(lo);
  *idx = t - (win_offset(cu, lo, n) / size + lo);
  return lo;
}

inline int win_tiles(int64_t n, int64_t size, int64_t batch) {
  return (int)(n / size + batch + 1);
}

// Consecutive work items on one XCD (workgroups go round the eight XCDs), so
// that neighbouring tiles find each other's keys in its L2.
__device__ inline int win_item() {
  const int per = gridDim.x / NXCD;  // the host rounds the grid up to NXCD
  return ((int)blockIdx.x % NXCD) * per + (int)blockIdx.x / NXCD;
}
inline int win_grid(int64_t items) { return (int)((items + NXCD - 1) / NXCD * NXCD); }

// Bias of a tile's relative positions: the 2 R + 1 values and WIN_PAD copies
// of the end values on both sides, in log2 units.  A tile of 64 keys and 32
// queries that has any position inside (-R, R) stays within the padding, so
// its elements are read at constant offsets from one address.
constexpr int WIN_PAD = 96;
__host__ __device__ inline int win_bias_len(int range) { return 2 * range + 1 + 2 * WIN_PAD; }

template <int DT>
__device__ inline float win_bias_at(const WinArgs& a, int head, int m) {
  int b = a.buckets[m];
  b = b < 0 ? 0 : (b >= a.n_buckets ? a.n_buckets - 1 : b);
  const float x = to_f32<DT>(a.table[(int64_t)b * a.hq + head]);
  return x < WIN_MASKED ? -__builtin_inf() : x * 1.4426950408889634f;
}

// The padded bias of `heads` consecutive heads, by 256 threads: the buckets of a
// thread's positions are read at once, then the table's entries, so that the
// two dependent reads are paid once and not for every position.
template <int DT>
__device__ inline void win_load_bias(const WinArgs& a, int head, int heads, float* dst, int tid) {
  constexpr int MOST = (2 * WIN_MAX_RANGE + 1 + 2 * WIN_PAD + 255) / 256;
  const int n = win_bias_len(a.range), top = 2 * a.range;
  int bucket[MOST];
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    const int i = tid + u * 256;
    bucket[u] = 0;
    if (i < n) {
      int m = i - WIN_PAD;
      m = m < 0 ? 0 : (m > top ? top : m);
      const int b = a.buckets[m];
      bucket[u] = b < 0 ? 0 : (b >= a.n_buckets ? a.n_buckets - 1 : b);
    }
  }
  for (int h = 0; h < heads; ++h)
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      const int i = tid + u * 256;
      if (i < n) {
        const float x = to_f32<DT>(a.table[(int64_t)bucket[u] * a.hq + head + h]);
        dst[h * n + i] = x < WIN_MASKED ? -__builtin_inf() : x * 1.4426950408889634f;
      }
    }
}

// The backward subtracts rowsum(dO * O) from dP.  With O as rounded to 16 bits
// that costs the gradients precision where a row sees few keys (dQ off by 2.55e-3
// in the 2-norm, not 2.38e-3, of which the roundings of dS and of dQ itself are
// 2.35e-3).  So a forward that will be followed by a backward also stores the 8
// bits that come next: the bits of x in 32 less those of its rounding.  The
// forward and the kernel that reads them take 314 us for it, not 302 (32768
// tokens, 16 heads of 64, windows of 511; 2% at windows of 1024).
template <int DT>
constexpr int LOW_SHIFT = DT == LSRM_BF16 ? 8 : 5;  // of the 16 or 13 bits that rounding takes
template <int DT>
__device__ inline int low_part(float x, uint32_t hi) {  // hi: x as stored (see stored_bits)
  constexpr int TOP = 128 << LOW_SHIFT<DT>;
  const int d = (int)__builtin_bit_cast(uint32_t, x) -
                (int)__builtin_bit_cast(uint32_t, to_f32<DT>((uint16_t)hi));
  return d < -TOP ? -TOP : (d > TOP - 1 ? TOP - 1 : d);
}
// The bytes of four elements in one word.
template <int DT>
__device__ inline uint32_t low_word(const float* x, uint32_t hi01, uint32_t hi23) {
  constexpr int S = LOW_SHIFT<DT> % 8;  // bf16: the second byte as it is
  constexpr uint32_t SEL = DT == LSRM_BF16 ? 0x0c0c0501u : 0x0c0c0400u;
  const uint32_t a =
      __builtin_amdgcn_perm((uint32_t)(low_part<DT>(x[1], hi01 >> 16) >> S),
                            (uint32_t)(low_part<DT>(x[0], hi01 & 0xffffu) >> S), SEL);
  const uint32_t b =
      __builtin_amdgcn_perm((uint32_t)(low_part<DT>(x[3], hi23 >> 16) >> S),
                            (uint32_t)(low_part<DT>(x[2], hi23 & 0xffffu) >> S), SEL);
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
template <int DT>
__device__ inline float with_low(uint16_t hi, int low) {
  return __builtin_bit_cast(
      float, (uint32_t)((int)__builtin_bit_cast(uint32_t, to_f32<DT>(hi)) +
                        low * (1 << LOW_SHIFT<DT>)));
}
// The compiler turns a product and its rounding to fp16 into one instruction that
// rounds once, for some of a value's uses and not for others: two numbers where
// the code has one.  What is stored and what is read back are the same from here.
__device__ inline uint32_t stored_bits(uint32_t w) {
  asm("" : "+v"(w));
  return w;
}
// Where column c of a row has its byte: the columns that a lane of one half of a
// wave reads (eight of every sixteen) lie together.
template <int D>
__device__ inline int low_at(int c) {
  return (c >> 3 & 1) * (D / 2) + (c >> 4) * 8 + (c & 7);
}

// Bits lo .. hi - 1 of 32 (any lo and hi).
__device__ inline uint32_t bits_below(int n) {
  n = n < 0 ? 0 : (n > 32 ? 32 : n);
  return (uint32_t)(0xffffffffull >> (32 - n));
}
__device__ inline uint32_t bits_between(int lo, int hi) {
  return bits_below(hi) & ~bits_below(lo);
}
// Element v of an accumulator (its lane's row acc_row(v, 0)): the value where
// its bit of the mask is set, else `other`; two instructions and no branch.
__device__ inline float keep(uint32_t mask, int v, float x, float other) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)mask, acc_row(v, 0), 1);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) |
                                       (__builtin_bit_cast(uint32_t, other) & ~m));
}

// x of the lanes 0 - 31, then y of the lanes 0 - 31: the first result; x of the
// lanes 32 - 63, then y of those: the second.
__device__ inline void swap_halves(uint32_t& x, uint32_t& y) {
  const auto sw = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = (uint32_t)sw[0];
  y = (uint32_t)sw[1];
}
// Both halves of a wave: the value of lane l ^ 32 combined with this lane's.
__device__ inline float half_max(float m) {
  const auto sw = __builtin_amdgcn_permlane32_swap(
      __builtin_bit_cast(unsigned, m), __builtin_bit_cast(unsigned, m), false, false);
  return __builtin_elementwise_maximum(__builtin_bit_cast(float, (unsigned)sw[0]),
                                       __builtin_bit_cast(float, (unsigned)sw[1]));
}
__device__ inline float half_sum(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(
      __builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, (unsigned)sw[0]) + __builtin_bit_cast(float, (unsigned)sw[1]);
}

// 16 channels of the accumulators' rows (values 8 i .. of a lane: four of every
// eight channels), times f, in 16 bits: eight consecutive channels a lane, the
// first half's lanes with the lower ones.  All lanes take part.
template <int DT>
__device__ inline u32x4 row_piece(const f32x16& x, int i, float f) {
  uint32_t w0 = pack2<DT>(x[8 * i] * f, x[8 * i + 1] * f);
  uint32_t w1 = pack2<DT>(x[8 * i + 2] * f, x[8 * i + 3] * f);
  uint32_t w2 = pack2<DT>(x[8 * i + 4] * f, x[8 * i + 5] * f);
  uint32_t w3 = pack2<DT>(x[8 * i + 6] * f, x[8 * i + 7] * f);
  swap_halves(w0, w2);
  swap_halves(w1, w3);
  return u32x4{w0, w1, w2, w3};
}

// A wave-uniform address in scalar registers.
__device__ inline const uint16_t* uniform_ptr(const uint16_t* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint16_t*>(
      ((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}

// Copies of NR-row tiles of one head into LDS, all four waves.  The lane's
// offsets within a full tile are kept; a tile of cnt < NR rows reads its last
// row in place of the missing ones.
template <int D, int NR>
struct TileCopy {
  using G = KvTile<D, NR>;
  uint32_t off[G::LPW];
  uint32_t row_bytes;
  __device__ inline void init(int64_t stride, int wv, int lane) {
    row_bytes = (uint32_t)stride * 2;
#pragma unroll
    for (int j = 0; j < G::LPW; ++j) {
      const int row = (wv * G::LPW + j) * G::KPL + lane / G::CH;
      off[j] = (uint32_t)row * row_bytes + (((lane % G::CH) ^ G::swz(row)) << 4);
    }
  }
  __device__ inline __attribute__((always_inline)) void copy(const uint16_t* base, int cnt,
                                                             char* dst, int wv, int lane) const {
    const uint32_t d0 = (uint32_t)uniform((int)(lds_addr(dst) + wv * G::LPW * 1024));
    base = uniform_ptr(base);
    if (cnt >= NR) {
#pragma unroll
      for (int j = 0; j < G::LPW; ++j) copy16_to_lds(base, off[j], d0 + j * 1024);
    } else {
#pragma unroll
      for (int j = 0; j < G::LPW; ++j) {
        const int row = (wv * G::LPW + j) * G::KPL + lane / G::CH;
        const int over = row < cnt ? 0 : row - (cnt - 1);
        copy16_to_lds(base, off[j] - (uint32_t)over * row_bytes, d0 + j * 1024);
      }
    }
  }
};

// Largest of N values, three at a time (v_maximum3_f32).
template <int N>
__device__ inline float max_of(const float* x) {
  if constexpr (N == 1) {
    return x[0];
  } else {
    float t[(N + 2) / 3];
#pragma unroll
    for (int i = 0; i < (N + 2) / 3; ++i) {
      t[i] = x[3 * i];
      if (3 * i + 1 < N) t[i] = __builtin_elementwise_maximum(t[i], x[3 * i + 1]);
      if (3 * i + 2 < N) t[i] = __builtin_elementwise_maximum(t[i], x[3 * i + 2]);
    }
    return max_of<(N + 2) / 3>(t);
  }
}

// 64 floats, lane l's at base + min(l, cnt - 1), to LDS; one wave.
__device__ inline void win_copy_floats(const float* base, int cnt, float* dst, int lane) {
  const int from = lane < cnt ? lane : cnt - 1;
  const float* b = reinterpret_cast<const float*>(
      uniform_ptr(reinterpret_cast<const uint16_t*>(base)));
  const uint32_t d0 = (uint32_t)uniform((int)lds_addr(dst));
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dword %0, %1"
      :
      : "v"((uint32_t)from * 4u), "s"(b), "s"(d0)
      : "memory");
}

// Transposed MFMA operand: columns d (32 of block db) of rows k0 .. of a tile,
// in the slot order of the score accumulators (see KvTile).
template <int D>
struct TransposedRead {
  uint32_t off[D / 32][2];
  __device__ inline void init(int lane) {
    using G = KvTile<D>;
    const int hb = lane >> 5, gi = lane & 15, dh = (lane >> 4) & 1;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int dcol = db * 32 + dh * 16 + (gi & 3) * 4;
      const int k0 = hb * 4 + (gi >> 2);
      const int cb = dcol >> 3, half = (dcol & 4) * 2;
      off[db][0] = (uint32_t)(G::off(k0, cb) + half);
      off[db][1] = (uint32_t)(G::off(k0 + 8, cb) + half);
    }
  }
  // Rows row16 .. row16 + 15 (a multiple of 16).
  __device__ inline u32x4 read(const char* tile, int db, int row16) const {
    const int o = row16 * (D * 2);
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(tile + o + off[db][0])));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(tile + o + off[db][1])));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

}  // namespace lsrm
