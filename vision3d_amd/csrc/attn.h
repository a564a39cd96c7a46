// attn.h -- what the attention kernels share: arguments, the way from a workgroup to its sequence, tiles in LDS and the
// matrix instructions' operands.
#ifndef V3D_CSRC_ATTN_H_
#define V3D_CSRC_ATTN_H_

#include "common.h"
#include "numeric.h"

namespace v3d {

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__host__ __device__ constexpr int attn_pow2(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

constexpr int kAttnWaves = 4;
constexpr int kAttnRows = 32 * kAttnWaves;  // rows (or keys) of a workgroup's tile
constexpr int kAttnWalk = 256;              // sequences that every wave looks through by itself, see locate

// Element strides throughout.  Rows of the keys: row j of sequence b is at (first row of b + j) * row stride in a pack,
// at b * batch stride + j * row stride in a cache (`capacity` > 0).
struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;                 // (total_q, H, D) contiguous
  void* rest;                // what rounding took from out, in its type (16-bit types, for the backward); or NULL
  float* lse;                // (total_q, H) log2 of the sum of exponentials, -inf for a row without keys; or NULL
  const int64_t* q_lengths;  // (B), NULL in a cache: every sequence has `tokens` queries
  const int64_t* s_lengths;  // (B)
  const int64_t* table;      // a pack of more than kAttnWalk sequences: (3 or 4, B + 1), see attn_table_launch
  int64_t total_q, total_s;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, k_batch, v_batch;
  int64_t capacity;
  int tokens;
  int B, H, KV, G, D;        // G = H / KV query heads share a key head
  unsigned g_mul, g_shift;   // n / G = mulhi(n, g_mul) >> g_shift for n < 2^31 (G > 1)
  float scale;
  int causal;
  int splits;                // parts that the keys of a row tile are divided into
  float* part_o;             // splits > 1: (tile, KV, split, rows of a tile, D) unnormalised rows ...
  float* part_ml;            // ... and (tile, KV, split, rows of a tile, 2): maximum (of q . k) and sum
};

__device__ __forceinline__ int div_g(const AttnArgs& a, int n) {
  return a.G == 1 ? n : (int)(__umulhi((unsigned)n, a.g_mul) >> a.g_shift);
}

// A workgroup's sequence.  All fields are wave-uniform.
struct AttnSeq {
  int b = 0;
  int tile = 0;              // row tile (or key tile) inside the sequence
  bool found = false;
  int64_t q_off = 0, s_off = 0;
  int q_len = 0, s_len = 0;
  int64_t spare = 0;         // !found: how many tiles past the last one
  int64_t q_end = 0, s_end = 0;  // !found: rows that belong to a sequence
};

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t hi) { return v < 0 ? 0 : (v < hi ? v : hi); }

__device__ __forceinline__ int64_t lanes_prefix(int64_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

template <int N>
struct Const {
  static constexpr int value = N;
};

__device__ __forceinline__ int wave_sum(int x) {
  auto dpp = [](int v, auto ctrl) { return __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, 0xf, 0xf, true); };
  x += dpp(x, Const<0xB1>{});   // quad_perm [1,0,3,2]
  x += dpp(x, Const<0x4E>{});   // quad_perm [2,3,0,1]
  x += dpp(x, Const<0x141>{});  // row_half_mirror
  x += dpp(x, Const<0x140>{});  // row_mirror
  return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) +
         __builtin_amdgcn_readlane(x, 48);
}

// Tile number `t` of the pack: sequence b has ceil(rows_b / TILE) tiles, rows_b = q_len * G (BY_KEYS: s_len).  The lengths
// are device data, so the launch covers the bound total / TILE + B and the kernels look their sequence up here: every wave
// by itself, one lane per sequence (or a few), no LDS and no barrier.  Negative lengths count as 0; lengths that overrun the
// totals are cut, so that no row outside the buffers is ever addressed.
//
// That every wave adds all lengths up costs the square of their number, so more than kAttnWalk sequences are looked up in a table
// of the rows and tiles before each, which a small kernel writes first: 64 places of it at a time, two steps for 4096 sequences.
// Sequences of 4 tokens, 8 heads of 32, bf16, forward, without and with the table: 128 sequences 15 / 22 us, 256 22 / 24, 512 45 /
// 38, 1024 155 / 64, 16384 32000 / 980 us.
//
// The causal tiles of up to 64 sequences are numbered by work, the most first, whatever sequence they lie in: a row tile's
// work grows with its place in the sequence, a key tile's with its distance from the end, so the numbering goes level by
// level, from the last tiles of the longest sequence down to the first tiles of all (8192 tokens in 5 sequences, 16/4 heads of
// 128, bf16: forward 140 -> 111 us, dq 146 -> 130 us).  Without a mask, and with more sequences, tiles are numbered one
// sequence after another, so that those which share keys and values run together (32 pairs of 512 tokens: 73 us against 78).
template <int TILE, bool BY_KEYS>
__device__ __forceinline__ AttnSeq locate(const AttnArgs& a, int64_t t) {
  const int lane = threadIdx.x & 63;
  AttnSeq r;
  auto tiles = [&](int64_t q, int64_t s) -> int64_t { return ((BY_KEYS ? s : q * a.G) + TILE - 1) / TILE; };
  auto len_q = [&](int i) { return clamp64(a.q_lengths[i], a.total_q); };
  auto len_s = [&](int i) { return clamp64(a.s_lengths[i], a.total_s); };
  if (a.B <= 64) {
    int64_t q = lane < a.B ? len_q(lane) : 0, s = lane < a.B ? len_s(lane) : 0;
    const int64_t iq = lanes_prefix(q, lane), is = lanes_prefix(s, lane);
    const int64_t q0 = clamp64(iq - q, a.total_q), s0 = clamp64(is - s, a.total_s);
    q = clamp64(q, a.total_q - q0);
    s = clamp64(s, a.total_s - s0);
    const int n = (int)tiles(q, s);
    const int all = wave_sum(n);
    if (t >= all) {
      r.spare = t - all;
      r.q_end = clamp64(__shfl(iq, 63, 64), a.total_q);
      r.s_end = clamp64(__shfl(is, 63, 64), a.total_s);
      return r;
    }
    if (!a.causal) {
      int pn = n;  // inclusive
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(pn, d, 64);
        if (lane >= d) pn += o;
      }
      const int src = __builtin_ctzll(__ballot(pn > (int)t));
      r.found = true;
      r.b = src;
      r.tile = (int)t - __shfl(pn - n, src, 64);
      r.q_off = __shfl(q0, src, 64);
      r.s_off = __shfl(s0, src, 64);
      r.q_len = (int)__shfl(q, src, 64);
      r.s_len = (int)__shfl(s, src, 64);
      return r;
    }
    // the highest level of which some tile is still ahead of number t: tiles at level l or above > t
    int level = 0, above = 0;
    if (a.B == 1) {
      level = all - 1 - (int)t;
    } else {
      int most = n;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) most = max(most, __shfl_xor(most, d, 64));
      int low = 0, high = __builtin_amdgcn_readfirstlane(most);  // count(low) > t >= count(high)
      while (high - low > 1) {
        const int mid = (low + high) >> 1, count = wave_sum(max(0, n - mid));
        if (count > (int)t) {
          low = mid;
        } else {
          high = mid;
          above = count;
        }
      }
      level = low;
    }
    const uint64_t mask = __ballot(n > level);
    const int rank = __builtin_popcountll(mask & (((uint64_t)1 << lane) - 1));
    const int src = a.B == 1 ? 0 : __builtin_ctzll(__ballot(n > level && rank == (int)t - above));
    r.found = true;
    r.b = src;
    r.tile = BY_KEYS ? __shfl(n, src, 64) - 1 - level : level;
    r.q_off = __shfl(q0, src, 64);
    r.s_off = __shfl(s0, src, 64);
    r.q_len = (int)__shfl(q, src, 64);
    r.s_len = (int)__shfl(s, src, 64);
    return r;
  }
  if (a.B <= kAttnWalk) {
    static_assert(kAttnWalk <= 64 * 64, "a lane's sequences are looked at by one wave at once");
    const int per = (a.B + 63) >> 6;
    int64_t sq = 0, ss = 0, st = 0;
    for (int e = 0; e < per; ++e) {
      const int i = lane * per + e;
      if (i < a.B) {
        const int64_t q = len_q(i), s = len_s(i);
        sq += q;
        ss += s;
        st += tiles(q, s);
      }
    }
    const int64_t iq = lanes_prefix(sq, lane), is = lanes_prefix(ss, lane), it = lanes_prefix(st, lane);
    const int64_t all = uniform64(__shfl(it, 63, 64));  // uniform to the compiler: what follows stays in scalar registers
    if (t >= all) {
      r.spare = t - all;
      r.q_end = clamp64(__shfl(iq, 63, 64), a.total_q);
      r.s_end = clamp64(__shfl(is, 63, 64), a.total_s);
      return r;
    }
    const int src = __builtin_ctzll(__ballot(it > t));  // the first lane whose tiles reach past t
    int64_t q0 = __shfl(iq - sq, src, 64), s0 = __shfl(is - ss, src, 64), t0 = __shfl(it - st, src, 64);
    const int i = src * per + lane;  // among that lane's sequences
    const bool in = lane < per && i < a.B;
    const int64_t q = in ? len_q(i) : 0, s = in ? len_s(i) : 0, n = in ? tiles(q, s) : 0;
    const int64_t pq = lanes_prefix(q, lane), ps = lanes_prefix(s, lane), pt = lanes_prefix(n, lane);
    const int at = __builtin_ctzll(__ballot(t0 + pt > t));
    q0 = clamp64(q0 + __shfl(pq - q, at, 64), a.total_q);
    s0 = clamp64(s0 + __shfl(ps - s, at, 64), a.total_s);
    r.found = true;
    r.b = src * per + at;
    r.tile = (int)(t - t0 - __shfl(pt - n, at, 64));
    r.q_off = q0;
    r.s_off = s0;
    r.q_len = (int)clamp64(__shfl(q, at, 64), a.total_q - q0);
    r.s_len = (int)clamp64(__shfl(s, at, 64), a.total_s - s0);
    return r;
  }
  const int64_t n = a.B + 1;
  const int64_t* before = a.table + (BY_KEYS ? 3 : 2) * n;  // tiles before a sequence
  const int64_t all = uniform64(before[a.B]);
  if (t >= all) {
    r.spare = t - all;
    r.q_end = a.table[a.B];
    r.s_end = a.table[n + a.B];
    return r;
  }
  int low = 0, high = a.B;  // before[low] <= t < before[high]
  while (high - low > 1) {
    const int step = (high - low + 63) >> 6;
    const int at = (int)min((int64_t)high, low + (int64_t)(lane + 1) * step);  // the last lane's is `high`
    const int src = __builtin_ctzll(__ballot(before[at] > t));
    high = (int)min((int64_t)high, low + (int64_t)(src + 1) * step);
    low += src * step;
  }
  r.found = true;
  r.b = low;
  r.tile = (int)(t - before[low]);
  r.q_off = a.table[low];
  r.s_off = a.table[n + low];
  r.q_len = (int)(a.table[low + 1] - r.q_off);
  r.s_len = (int)(a.table[n + low + 1] - r.s_off);
  return r;
}

// The same for a cache: the geometry is known on the host, only the filled length is read.
template <int TILE>
__device__ __forceinline__ AttnSeq locate_cache(const AttnArgs& a, int64_t t) {
  AttnSeq r;
  const int per = (int)(((int64_t)a.tokens * a.G + TILE - 1) / TILE);
  r.b = (int)(t / per);
  r.tile = (int)(t % per);
  r.found = r.b < a.B;
  if (!r.found) return r;
  r.q_off = (int64_t)r.b * a.tokens;
  r.q_len = a.tokens;
  r.s_len = (int)uniform64(clamp64(a.s_lengths[r.b], a.capacity));
  return r;
}

// (The fields once more through readfirstlane: descriptors and loop bounds that the compiler cannot prove uniform cost a
// loop per load.)
__device__ __forceinline__ AttnSeq uniform(AttnSeq r) {
  r.b = __builtin_amdgcn_readfirstlane(r.b);
  r.tile = __builtin_amdgcn_readfirstlane(r.tile);
  r.found = __builtin_amdgcn_readfirstlane((int)r.found) != 0;
  r.q_off = uniform64(r.q_off);
  r.s_off = uniform64(r.s_off);
  r.q_len = __builtin_amdgcn_readfirstlane(r.q_len);
  r.s_len = __builtin_amdgcn_readfirstlane(r.s_len);
  r.spare = uniform64(r.spare);
  r.q_end = uniform64(r.q_end);
  r.s_end = uniform64(r.s_end);
  return r;
}

template <int TILE>
__device__ __forceinline__ AttnSeq locate_rows(const AttnArgs& a, int64_t t) {
  return uniform(a.capacity > 0 ? locate_cache<TILE>(a, t) : locate<TILE, false>(a, t));
}
template <int TILE>
__device__ __forceinline__ AttnSeq locate_keys(const AttnArgs& a, int64_t t) {
  return uniform(locate<TILE, true>(a, t));
}

// ---- numbers of the products -------------------------------------------------------------------------------------------
// 16-bit types go into the matrix instructions as they are (exact products, fp32 sums).  An fp32 number goes in as three bf16
// numbers that add up to it exactly (8 + 8 + 8 bits, cut off, so nothing overflows), and a product of two as the six of the
// nine partial products that reach 2^-24 of it: the same accuracy as fp32 products in 6 x 32 cycles where the fp32
// matrix instruction takes 8 x 64.  An infinity among fp32 inputs
// becomes a NaN where it is seen.
template <typename T>
struct Kind {
  typedef T U;                     // what lies in LDS and goes into the instructions
  static constexpr int P = 1;      // how many of them make a number
};
template <>
struct Kind<float> {
  typedef bf16 U;
  static constexpr int P = 3;
};

template <typename U>
struct Vec8;
template <>
struct Vec8<bf16> {
  typedef bf16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Vec8<f16> {
  typedef f16 type __attribute__((ext_vector_type(8)));
};

// An operand: 8 numbers of a lane.
template <typename T>
struct Op {
  typename Vec8<typename Kind<T>::U>::type part[Kind<T>::P];
};

template <typename T>
__device__ __forceinline__ float number(const Op<T>& op, int j) {
  float x = 0.f;
#pragma unroll
  for (int p = Kind<T>::P - 1; p >= 0; --p) x += to_f32(op.part[p][j]);  // exact
  return x;
}

__device__ __forceinline__ Op<float> split8(const float (&x)[8]) {
  unsigned word[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned a[3], b[3];
    float x0 = x[2 * j], x1 = x[2 * j + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      a[p] = __float_as_uint(x0);
      b[p] = __float_as_uint(x1);
      x0 -= __uint_as_float(a[p] & 0xffff0000u);
      x1 -= __uint_as_float(b[p] & 0xffff0000u);
      word[p][j] = __builtin_amdgcn_perm(b[p], a[p], 0x07060302u);  // the upper halves
    }
  }
  Op<float> op;
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const u32x4 w = {word[p][0], word[p][1], word[p][2], word[p][3]};
    op.part[p] = __builtin_bit_cast(Vec8<bf16>::type, w);
  }
  return op;
}

// ---- loads -------------------------------------------------------------------------------------------------------------
// Loads go through a buffer descriptor: what lies past its range comes back as zeros without a branch, so all loads of a
// tile are under way together.  Columns from D on are zeros too: 16 bytes past D are placed out of any range, 16 bytes that
// D ends inside are read up to D and shifted into place (hence a head of at least 16 bytes).
constexpr int kOutOfRange = 0x7fffffff;

__device__ __forceinline__ u32x4 load_buffer(const void* base, int bytes, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000),
                                               offset, 0, 0);
}

// 8 numbers as they come from memory.
template <typename T>
struct Raw {
  static constexpr int L = (int)sizeof(T) / 2;      // 16-byte loads
  static constexpr int E = 16 / (int)sizeof(T);     // numbers of a load
  u32x4 c[L];

  // Columns [col, col + 8) of a row that starts at element `at` from `base`; `there` false: zeros.
  __device__ __forceinline__ void load(const T* base, int bytes, int at, int col, int D, bool there) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const int c0 = col + l * E;
      c[l] = load_buffer(base, bytes, !there || c0 >= D ? kOutOfRange : (at + min(c0, D - E)) * (int)sizeof(T));
    }
  }
  __device__ __forceinline__ Op<T> op(int col, int D) const {
    u32x4 v[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      v[l] = c[l];
      if (D % E != 0) {
        asm volatile("" : "+v"(v[l]));  // stays a branch: as selects the shift would cost every tile of every head size
        const int c0 = col + l * E, by = c0 < D ? max(0, c0 + E - D) : 0;
        unsigned __int128 x = __builtin_bit_cast(unsigned __int128, v[l]);
        x >>= by * 8 * (int)sizeof(T);
        v[l] = __builtin_bit_cast(u32x4, x);
      }
    }
    if constexpr (L == 1) {
      Op<T> r;
      r.part[0] = __builtin_bit_cast(typename Vec8<T>::type, v[0]);
      return r;
    } else {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(v[j / 4][j % 4]);
      return split8(x);
    }
  }
  __device__ __forceinline__ bool nonfinite() const {
    bool bad = false;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const Packed<T, E> v = __builtin_bit_cast(Packed<T , E>, c[l]);
#pragma unroll
      for (int j = 0; j < E; ++j) bad |= !(__builtin_fabsf(to_f32(v.v[j])) < __builtin_inff());
    }
    return bad;
  }
};

// The operands of all product steps over the head size from one row in memory: `at` = this lane's row in elements from
// `base` (wave-uniform).
template <typename T, int STEPS>
__device__ __forceinline__ void load_ops(Op<T> (&op)[STEPS], const T* base, int at, int half, int D, bool there) {
  Raw<T> raw[STEPS];
#pragma unroll
  for (int st = 0; st < STEPS; ++st) raw[st].load(base, kOutOfRange, at, st * 16 + 8 * half, D, there);
#pragma unroll
  for (int st = 0; st < STEPS; ++st) op[st] = raw[st].op(st * 16 + 8 * half, D);
}

// `x`, such that what is computed from it is computed again in every turn of a loop (kAgain).  The compiler otherwise computes
// the LDS addresses of a tile once, before the loop, and keeps them all: with fp32 heads past 192 that is more registers than
// are left, and an address read back from memory costs more than its few instructions (where `x` is masked afterwards, so that
// its range is known: 134 -> 80 instructions a chunk).
template <bool kAgain>
__device__ __forceinline__ int again(int x) {
  if constexpr (kAgain) asm volatile("" : "+v"(x));
  return x;
}

// The operands of all product steps over the head size that a wave uses in its loop: kept in registers, but fp32 heads past 128
// are read again from the cache where they are used, kAhead steps ahead, and split there: beside the sums there is no room (48 to
// 173 registers spilled).  Training in fp32, 8 heads, 8 sequences of 500 tokens: heads of 256 2405 -> 1415 us, of 160 1155 -> 1016;
// 1, 3, 4 and 8 steps ahead 1590, 1560, 1590 and 1690 for 1545 us (before the addresses of `again`).
template <typename T, int HD>
struct Held {
  static constexpr int STEPS = HD / 16;
  static constexpr int kAhead = 2;
  static constexpr bool kLate = Kind<T>::P == 3 && HD > 128;
  Op<T> ops[kLate ? 1 : STEPS];
  Raw<T> raw[kLate ? kAhead : 1];
  const T* base;
  int at, half, D;
  bool there;

  __device__ __forceinline__ void load(const T* from, int row, int h, int d, bool in) {
    base = from;
    at = row;
    half = h;
    D = d;
    there = in;
    if constexpr (!kLate) load_ops<T>(ops, from, row, half, D, in);
  }
  // Before the steps of a turn of the loop.
  __device__ __forceinline__ void begin() {
    if constexpr (kLate) {
      at = again<true>(at);
#pragma unroll
      for (int st = 0; st < kAhead; ++st) raw[st].load(base, kOutOfRange, at, st * 16 + 8 * half, D, there);
    }
  }
  // The operand of step st, in order.
  __device__ __forceinline__ Op<T> get(int st) {
    if constexpr (kLate) {
      const Op<T> op = raw[st % kAhead].op(st * 16 + 8 * half, D);
      if (st + kAhead < STEPS) raw[st % kAhead].load(base, kOutOfRange, at, (st + kAhead) * 16 + 8 * half, D, there);
      return op;
    } else {
      return ops[st];
    }
  }
};

// ---- tiles in LDS ------------------------------------------------------------------------------------------------------
// A tile is P planes of ROWS rows of HDP 16-bit numbers (the head size rounded up to a power of two), moved in chunks of 8.
// It is read in two ways: 16 consecutive rows at one chunk (read_cols), and 4 consecutive rows at 64 consecutive bytes
// (read_rows).  Chunks sit at their column XOR f(row), f chosen so that both ways touch each of the 64 banks once: f takes
// 16 values over 16 rows that start a bank line, and its bits that move 64 bytes change between consecutive rows.
template <int HDP>
__device__ __forceinline__ int place(int row, int chunk) {
  constexpr int CPR = HDP / 8;
  if constexpr (CPR >= 16) return chunk ^ (((row & 3) << 2) | ((row >> 2) & 3));
  if constexpr (CPR == 8) return chunk ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
  return chunk ^ ((row >> 2) & 3);
}

// Offset of element `col` of `row` in a plane.
template <int HDP>
__device__ __forceinline__ int tile_at(int row, int col) {
  return row * HDP + place<HDP>(row, col / 8) * 8 + col % 8;
}

// A tile on its way from memory to LDS in the registers of THREADS threads.
template <typename T, int HD, int ROWS, int THREADS, int PLANE = ROWS>  // PLANE: rows of a plane of the tile
struct TileStage {
  typedef typename Kind<T>::U U;
  static constexpr int CPR = HD / 8;                // chunks of a row
  static constexpr int CH = (ROWS * CPR + THREADS - 1) / THREADS;
  static constexpr bool kEven = ROWS * CPR % THREADS == 0;  // else the last chunk of some threads repeats the last row's
  Raw<T> c[CH];

  static constexpr bool kTight = Kind<T>::P == 3 && HD > 192;  // registers are short
  static constexpr bool kFixed = THREADS % CPR == 0;          // a thread stays with one column
  static __device__ __forceinline__ int thread() { return again<kTight>((int)threadIdx.x) & (THREADS - 1); }
  static __device__ __forceinline__ int row_of(int i) {
    const int row = kFixed ? i * (THREADS / CPR) + thread() / CPR : (i * THREADS + thread()) / CPR;
    return kEven ? row : min(row, ROWS - 1);
  }
  static __device__ __forceinline__ int col_of(int i) { return (kFixed ? thread() : i * THREADS + thread()) % CPR * 8; }

  // Rows [0, count) at `base`, `stride` elements apart (a tile spans less than 2^31 bytes); count <= 0: nothing is read.
  __device__ __forceinline__ void fetch(const T* base, int64_t stride, int D, int count) {
    const int bytes = count <= 0 ? 0 : ((min(count, ROWS) - 1) * (int)stride + D) * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < CH; ++i) c[i].load(base, bytes, row_of(i) * (int)stride, col_of(i), D, true);
  }
  // The same for rows at offsets of their own (elements, non-negative, below 2^29).
  template <typename Offset>
  __device__ __forceinline__ void fetch_rows(const T* base, Offset offset, int D, int count) {
#pragma unroll
    for (int i = 0; i < CH; ++i) c[i].load(base, kOutOfRange, offset(row_of(i)), col_of(i), D, row_of(i) < count);
  }
  __device__ __forceinline__ void store(U* tile, int D) const {
    constexpr int HDP = attn_pow2(HD);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if constexpr (kTight) __builtin_amdgcn_sched_barrier(0);  // one split at a time
      const Op<T> op = c[i].op(col_of(i), D);
#pragma unroll
      for (int p = 0; p < Kind<T>::P; ++p)
        *reinterpret_cast<typename Vec8<U>::type*>(tile + p * (PLANE * HDP) + tile_at<HDP>(row_of(i), col_of(i))) = op.part[p];
    }
  }
  __device__ __forceinline__ bool nonfinite() const {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < CH; ++i) bad |= c[i].nonfinite();
    return bad;
  }
};

// ---- matrix instructions -----------------------------------------------------------------------------------------------
// Everything is built on the 32 x 32 result layout: lane l holds column l % 32, register r holds row
// 8 (r / 4) + 4 (l / 32) + r % 4 (`acc_row`).  The scores are computed transposed (keys x queries): a lane owns ONE query,
// so its maximum, sum and rescaling are scalars of the lane, and the probabilities are the next product's operand in the
// registers where they were computed -- the keys of a product are summed in any order, so the values are read in the
// order in which the result layout holds the keys (no lane exchange in between).
__device__ __forceinline__ constexpr int acc_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

__device__ __forceinline__ f32x16 mfma(Vec8<bf16>::type a, Vec8<bf16>::type b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Vec8<f16>::type a, Vec8<f16>::type b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// c + a b over 16 summands (8 of each half of the lanes); fp32: the partial products from the small to the large.
template <typename T>
__device__ __forceinline__ f32x16 product(const Op<T>& a, const Op<T>& b, f32x16 c) {
  if constexpr (Kind<T>::P == 3) {
    c = mfma(a.part[0], b.part[2], c);
    c = mfma(a.part[2], b.part[0], c);
    c = mfma(a.part[1], b.part[1], c);
    c = mfma(a.part[0], b.part[1], c);
    c = mfma(a.part[1], b.part[0], c);
  }
  return mfma(a.part[0], b.part[0], c);
}

// The A operand of a product step whose summands are COLUMNS of the tile: row `row`, columns [16 step + 8 half, + 8).
template <typename T, int HDP, int ROWS>
__device__ __forceinline__ Op<T> read_cols(const typename Kind<T>::U* tile, int row, int step, int half) {
  typedef typename Kind<T>::U U;
  Op<T> op;
#pragma unroll
  for (int p = 0; p < Kind<T>::P; ++p)
    op.part[p] = *reinterpret_cast<const typename Vec8<U>::type*>(tile + p * (ROWS * HDP) +
                                                                  tile_at<HDP>(row, step * 16 + 8 * half));
  return op;
}

// The A operand of a product step whose summands are ROWS of the tile, in the order of the result layout: step u of a
// 32-row block covers registers [8 u, 8 u + 8) of that layout.  Lane l stands for column d0 + l % 32.  gfx950's transposing
// LDS read: 16 lanes read 4 rows x 16 columns (lane i: row i / 4, columns 4 (i % 4) ..), each is handed its column's 4 rows.
template <typename T, int HDP, int ROWS>
__device__ __forceinline__ Op<T> read_rows(const typename Kind<T>::U* tile, int row0, int u, int d0, int lane) {
  typedef typename Kind<T>::U U;
  const int i = lane & 15;
  const int half = lane >> 5;
  const int col = d0 + (lane & 16) + 4 * (i & 3);
  Op<T> op;
#pragma unroll
  for (int p = 0; p < Kind<T>::P; ++p) {
    union {
      s16x4 quad[2];
      typename Vec8<U>::type all;
    } r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + 16 * u + 8 * h + 4 * half + (i >> 2);
      U* at = const_cast<U*>(tile) + p * (ROWS * HDP) + tile_at<HDP>(row, col);
      r.quad[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)reinterpret_cast<s16x4*>(at));
    }
    op.part[p] = r.all;
  }
  return op;
}

// The result layout's registers [8 u, 8 u + 8) of a 32 x 32 block as the B operand that goes with read_rows.  16-bit types:
// rounded to the type, as the other factor is (half a step of each summand, of either sign: the matrix instruction takes two
// operands of one type, and 32-bit summands would cost three products or six).  In bf16 that is relative to the summand
// whatever its size; what fp16 is to hold is brought into its range first.
template <typename T>
__device__ __forceinline__ Op<T> pack_rows(const f32x16& x, int u) {
  if constexpr (Kind<T>::P == 3) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[u * 8 + j];
    return split8(v);
  } else {
    Op<T> op;
#pragma unroll
    for (int j = 0; j < 8; ++j) op.part[0][j] = from_f32<T>(x[u * 8 + j]);
    return op;
  }
}

constexpr float kLog2e = 1.44269504088896340736f;

// Over the two lanes (l, l + 32) of a column, without LDS.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32; 2^-inf = 0

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// 4 elements of a row from `col` on, as far as D goes.
template <typename T>
__device__ __forceinline__ void store4(T* row, int col, int D, const float (&v)[4]) {
  if (col + 4 <= D) {
    store_vec<T, 4>(row + col, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < D) row[col + j] = from_f32<T>(v[j]);
  }
}

// A result whose column is this lane's row and whose rows are the row's elements, times `f`, to memory.
template <typename T, int DT>
__device__ __forceinline__ void store_rows(T* row, const f32x16 (&acc)[DT], float f, int D, int half) {
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v[4] = {acc[d][g * 4] * f, acc[d][g * 4 + 1] * f, acc[d][g * 4 + 2] * f, acc[d][g * 4 + 3] * f};
      store4<T>(row, d * 32 + 8 * g + 4 * half, D, v);
    }
}

// The mask of a row: its token sees the keys [0, this).
__device__ __forceinline__ int attn_limit(const AttnArgs& a, const AttnSeq& seq, int token) {
  return a.causal ? max(0, min(seq.s_len, token + seq.s_len - seq.q_len + 1)) : seq.s_len;
}

// Host side: the heads, and the division by the group's size as a product (exact for 31-bit numerators: the multiplier is
// 2^(31 + s) / G rounded up with 2^s >= G, its excess times n stays below 2^(31 + s)).
inline void attn_heads(AttnArgs& a, int H, int KV, int D) {
  a.H = H;
  a.KV = KV;
  a.G = H / KV;
  a.D = D;
  unsigned s = 0;
  while (((int64_t)1 << s) < a.G) ++s;
  a.g_mul = s == 0 ? 0u : (unsigned)((((uint64_t)1 << (31 + s)) + a.G - 1) / a.G);
  a.g_shift = s == 0 ? 0u : s - 1;
}

// Host side: fills `a.table` (attention.hip): first rows of the queries' sequences, of the keys' and the row tiles before each, if
// key_tile > 0 the key tiles too; the last entry of each is the end of all.
inline size_t attn_table_bytes(int B, int rows) { return B > kAttnWalk ? align_up((size_t)rows * ((size_t)B + 1) * 8, 256) : 0; }
int attn_table_launch(AttnArgs& a, void* table, int row_tile, int key_tile, hipStream_t stream, const char* what);

// Host side: parts that a row tile's keys and a key tile's rows are divided into in the backward (attention_bwd.hip).
int attn_backward_q_splits(int dtype, int B, int64_t total_q, int64_t total_s, int KV, int G);
int attn_backward_splits(int B, int64_t total_s, int KV, int D);

constexpr int64_t kAttnMaxGroups = ((int64_t)1 << 24) - 1;  // a launch holds less than 2^32 threads, 256 a workgroup

// Host side: the argument checks of every entry point (attention.hip).
int attn_check(const char* what, int dtype, int B, int64_t total_q, int64_t total_s, int H, int KV, int D, float scale);
int attn_check_strides(const char* what, const AttnArgs& a);
// Host side: the smallest built head size that holds D, 0 if there is none.
inline int attn_head_size(int D) {
  for (int hd : {32, 64, 96, 128, 192, 256})
    if (D <= hd) return hd;
  return 0;
}

}  // namespace v3d

#endif
