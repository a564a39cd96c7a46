// attention.hip -- softmax attention inside the sequences of a pack, and of new tokens against cached keys and values.
//
//   s_ij = scale * q_i . k_j over the keys that query i sees,  o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// Rows: the G = H / KV query heads of a key head are folded into the rows of that head's products (row = token * G + head),
// so grouped heads read every key once per tile whatever G is, and a single token of 8 heads fills 8 columns of a product
// instead of one.
//
// Measured: causal prompt of 12288 tokens in 6 sequences, 32/8 heads of 128, bf16: 300 us = 790 TFLOP/s (296 to 315 us from card
// to card; matrix pipe 38 % busy, no bank conflicts; two waves a SIMD, bound by the exponentials and by the issue of both); 32
// pairs of 512 tokens, 4 heads of 64, fp32: 70 us = 112 TFLOP/s (the library's fp32 product: 153); 32 caches of 2048 ... 8192
// rows, one token, 32/8 heads of 128, bf16: 137 us = 4.6 TB/s.
#include <algorithm>

#include "attn.h"

namespace v3d {

__device__ __forceinline__ void wave_order() {  // LDS accesses of a wave stay in program order
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// fp16 keeps 11 bits down to 2^-14 and nothing below 2^-25, where a long cache still has weight (2^15 keys of 2^-25 are 2^-10 of
// the row).  The probabilities are formed 2^7 times as large (in the exponent): with the room that a stale maximum asks for, 2^15.
template <typename T>
constexpr float kProbLift = __is_same(T, f16) ? 7.f : 0.f;

// A probability of score s = q . k is 2^(c2 s - base), base = c2 m - kProbLift for the running maximum m and c2 = scale log2(e):
// one multiply-add.  The rounding of c2 m is the same for the whole row, but past 2^31 it alone leaves the exponent's range: from
// kProbLarge on a probability is 2^(c2 (s - m) + kProbLift).
constexpr float kProbLarge = 0x1p20f;
template <typename T>
__device__ __forceinline__ float prob_base(float m, float c2) {
  return (m == -__builtin_inff() ? 0.f : m) * c2 - kProbLift<T>;
}
// What probabilities relative to m count relative to `to` >= m.
template <typename T>
__device__ __forceinline__ float prob_weight(float m, float to, float c2) {
  const float from = prob_base<T>(m, c2), base = prob_base<T>(to, c2);
  const bool fits = __builtin_fabsf(from) < kProbLarge && __builtin_fabsf(base) < kProbLarge && m > -__builtin_inff();
  return to == -__builtin_inff() ? 1.f : exp2_fast(fits ? from - base : (m - to) * c2);
}

// What a wave carries through its keys: 32 rows, one per lane and half.
template <typename T, int HD, bool AGAIN>
struct AttnWave {
  typedef typename Kind<T>::U U;
  static constexpr int HDP = attn_pow2(HD);
  static constexpr int STEPS = HD / 16;  // product steps over the head size
  static constexpr int DT = HD / 32;
  static constexpr bool kAgain = AGAIN;  // see again()

  Held<T, HD> q;
  f32x16 o[DT];
  float m = -__builtin_inff(), l = 0.f;  // running maximum of the products q . k, the sum of the probabilities (see scores)
  float base = -kProbLift<T>;  // of m
  bool large = false;          // some base of the wave is beyond kProbLarge
  float c2;
  int lane, half;
  int row, token, head;
  int limit;        // this lane's query sees the keys [0, limit)
  int least, most;  // of the wave's first and last row; most = 0: the wave has no rows
  int D;

  // `row0`: the wave's first row in the sequence.
  __device__ __forceinline__ void begin(const AttnArgs& a, const AttnSeq& seq, int kvh, int row0, int rows, bool load_q) {
    D = a.D;
    lane = threadIdx.x & 63;
    half = lane >> 5;
    row = row0 + (lane & 31);
    token = div_g(a, min(row, rows - 1));
    const int g = min(row, rows - 1) - token * a.G;
    head = kvh * a.G + g;
    limit = attn_limit(a, seq, token);
    least = __builtin_amdgcn_readfirstlane(limit);
    most = row0 < rows ? attn_limit(a, seq, div_g(a, min(row0 + 31, rows - 1))) : 0;
    c2 = a.scale * kLog2e;
    const int token0 = div_g(a, min(row0, rows - 1));
    if (load_q)
      q.load(static_cast<const T*>(a.q) + (seq.q_off + token0) * a.q_row + (int64_t)kvh * a.G * a.q_head,
             (token - token0) * (int)a.q_row + g * (int)a.q_head, half, a.D, true);
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = zero16();
  }

  // s = 2^(score - m) of a tile of 32 NT keys from key0 on; m, l and o move on.
  // kTile: the wave's rows are the tile `rows` in LDS, else they are in q.
  template <int NT, bool kTile>
  __device__ __forceinline__ void scores(const U* k, const U* rows, int key0, f32x16 (&s)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = zero16();
    if constexpr (!kTile) q.begin();
    const int at = again<kAgain>(lane) & 31;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      Op<T> qs;
      if constexpr (kTile)
        qs = read_cols<T, HDP, 32>(rows, at, st, half);
      else
        qs = q.get(st);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        s[n] = product<T>(read_cols<T, HDP, 32 * NT>(k, n * 32 + at, st, half), qs, s[n]);
    }
    if (key0 + 32 * NT > least) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + n * 32 + acc_row(r, half) >= limit) s[n][r] = -__builtin_inff();
      }
    }
    // maximum of the lane, then with the lane that holds the other keys of this query
    float top = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
    top = halves_max(top);
    // The maximum moves only when a probability would exceed 2^8: what was summed is rescaled rarely, and a stale maximum
    // costs no accuracy (16-bit probabilities keep their relative precision, the sums are fp32).
    if (__any((top - m) * c2 > 8.f)) {
      const float m_new = fmaxf(m, top);
      const float alpha = prob_weight<T>(m, m_new, c2);
      m = m_new;
      base = prob_base<T>(m, c2);
      large = __any(__builtin_fabsf(base) >= kProbLarge);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    float from = base;
    if (large) {
      const float at = m == -__builtin_inff() ? 0.f : m;
      from = -kProbLift<T>;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] -= at;
    }
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = exp2_fast(fmaf(s[n][r], c2, -from));
        sum += s[n][r];
      }
    l += sum;
  }

  template <int NT>
  __device__ __forceinline__ void values(const U* v, const f32x16 (&s)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Op<T> p = pack_rows<T>(s[n], u);
        const int at = again<kAgain>(lane) & 63;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = product<T>(read_rows<T, HDP, 32 * NT>(v, n * 32, u, d * 32, at), p, o[d]);
      }
  }

  // An infinity or NaN among the values of a tile that some query sees in part must not reach the queries that do not see
  // it (0 * inf).  Key by key it is added to the queries that do -- `p` is 32 x 32 of LDS that is the wave's own --; the
  // tile's owner then clears it for the product.
  template <int NT>
  __device__ __forceinline__ void add_nonfinite(U* p, const U* v, int key0, const f32x16 (&s)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      wave_order();
#pragma unroll
      for (int r = 0; r < 16; ++r) p[acc_row(r, half) * 32 + (lane & 31)] = from_f32<U>(s[n][r]);
      wave_order();
#pragma unroll 1
      for (int key = 0; key < 32 && key0 + n * 32 + key < most; ++key) {
        const float pk = to_f32(p[key * 32 + (lane & 31)]);
        const bool seen = key0 + n * 32 + key < limit;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float w = 0.f;
#pragma unroll
            for (int i = 0; i < Kind<T>::P; ++i)
              w += to_f32(v[i * (32 * NT * HDP) + tile_at<HDP>(n * 32 + key, d * 32 + acc_row(r, half))]);
            if (seen && !(__builtin_fabsf(w) < __builtin_inff())) o[d][r] += pk * w;
          }
      }
    }
  }
};

template <typename U>
__device__ __forceinline__ void clear_nonfinite(U* tile, int count, int first, int step) {
  for (int i = first; i < count; i += step)
    if (!(__builtin_fabsf(to_f32(tile[i])) < __builtin_inff())) tile[i] = (U)0.f;
}

// 4 finished values of a row: rounded to the type and, for the backward, what the rounding took.
template <typename T>
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t row, int col, const float (&v)[4]) {
  store4<T>(static_cast<T*>(a.out) + row * a.D, col, a.D, v);
  if (sizeof(T) == 2 && a.rest != nullptr) {
    float left[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) left[j] = v[j] - to_f32(from_f32<T>(v[j]));
    store4<T>(static_cast<T*>(a.rest) + row * a.D, col, a.D, left);
  }
}
__device__ __forceinline__ float inverse_sum(float l) {
  return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no keys: zeros; a NaN stays a NaN
}
// log2 of the row's sum of exp(scale * q . k) from its maximal product and its sum of probabilities.
template <typename T>
__device__ __forceinline__ float log_sum(const AttnArgs& a, float m, float l) {
  return l == 0.f ? -__builtin_inff() : prob_base<T>(m, a.scale * kLog2e) + log2f(l);
}

// The launch covers a bound of the pack's tiles: the rest of it clears the rows behind the last sequence.
template <typename T, int TILE>
__device__ __forceinline__ void clear_behind(const AttnArgs& a, const AttnSeq& seq, int kvh) {
  const int64_t rows = (a.total_q - seq.q_end) * a.G;
  for (int i = threadIdx.x; i < TILE; i += blockDim.x) {
    const int64_t r = seq.spare * TILE + i;
    if (r >= rows) break;
    const int64_t at = (seq.q_end + r / a.G) * a.H + (int64_t)kvh * a.G + r % a.G;
    for (int d = 0; d < a.D; ++d) {
      static_cast<T*>(a.out)[at * a.D + d] = (T)0.f;
      if (a.rest) static_cast<T*>(a.rest)[at * a.D + d] = (T)0.f;
    }
    if (a.lse) a.lse[at] = -__builtin_inff();
  }
}

// ---- many rows: 128 of them share the tiles of keys and values ---------------------------------------------------------
// Keys of a tile; two tiles (one worked on, one arriving) of keys and values lie in at most 96 KiB of LDS where that fits:
// two workgroups a CU with 16-bit heads of up to 128.
template <typename T, int HD>
constexpr int attn_keys() { return Kind<T>::P == 1 && HD <= 128 ? 64 : 32; }
template <typename T, int HD>
constexpr int attn_buffers() { return Kind<T>::P == 3 && HD > 128 ? 1 : 2; }
template <typename T, int HD>
constexpr int attn_occupancy() { return HD <= (Kind<T>::P == 1 ? 128 : 64) ? 2 : 1; }  // waves per SIMD that the registers are kept for

template <typename T, int HD>
__global__ __launch_bounds__(256, (attn_occupancy<T, HD>())) void attn_forward_kernel(const AttnArgs a) {
  typedef typename Kind<T>::U U;
  constexpr int HDP = attn_pow2(HD);
  constexpr int BN = attn_keys<T, HD>();
  constexpr int NT = BN / 32;  // 32-key blocks of a tile
  constexpr int BUFS = attn_buffers<T, HD>();
  constexpr int SIZE = Kind<T>::P * BN * HDP;
  __shared__ __attribute__((aligned(16))) U lds_k[BUFS][SIZE];
  __shared__ __attribute__((aligned(16))) U lds_v[BUFS][SIZE];
  __shared__ int lds_bad[BUFS];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const int split = (int)(id % a.splits);
  id /= a.splits;
  const AttnSeq seq = locate_rows<kAttnRows>(a, id);
  if (!seq.found) {
    if (a.capacity == 0 && split == 0) clear_behind<T, kAttnRows>(a, seq, kvh);
    return;
  }
  const int rows = seq.q_len * a.G;
  const int row0 = seq.tile * kAttnRows;
  if (row0 >= rows) return;  // lengths that overrun the total were cut
  AttnWave<T, HD, false> w;
  w.begin(a, seq, kvh, row0 + wave * 32, rows, true);
  // the workgroup's first and last rows bound what it has to look at
  const int most = attn_limit(a, seq, div_g(a, min(row0 + kAttnRows - 1, rows - 1)));
  const int least = attn_limit(a, seq, div_g(a, row0));

  const int tiles = (most + BN - 1) / BN;
  const int per_split = (tiles + a.splits - 1) / a.splits;
  const int t_begin = split * per_split, t_end = min(tiles, t_begin + per_split);
  const T* k = static_cast<const T*>(a.k) + seq.b * a.k_batch + seq.s_off * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + seq.b * a.v_batch + seq.s_off * a.v_row + (int64_t)kvh * a.v_head;

  // The tile after the one that is worked on is on its way meanwhile: its keys under the scores, its values under the
  // values' product, through the same registers.
  TileStage<T, HD, BN, 256> stage;
  if (threadIdx.x < BUFS) lds_bad[threadIdx.x] = 0;
  auto fetch_k = [&](int t) { stage.fetch(k + (int64_t)t * BN * a.k_row, a.k_row, a.D, seq.s_len - t * BN); };
  auto fetch_v = [&](int t) { stage.fetch(v + (int64_t)t * BN * a.v_row, a.v_row, a.D, seq.s_len - t * BN); };
  auto place_v = [&](int t, int buf) {
    stage.store(lds_v[buf], a.D);
    if (t * BN + BN > least && stage.nonfinite()) lds_bad[buf] = t + 1;
  };
  auto work = [&](int t, auto buffer) {
    constexpr int buf = decltype(buffer)::value, other = BUFS - 1 - buf;
    const int key0 = t * BN;
    const bool active = key0 < w.most, more = t + 1 < t_end;
    f32x16 s[NT];
    if (more) fetch_k(t + 1);
    if (active) w.template scores<NT, false>(lds_k[buf], nullptr, key0, s);
    if (key0 + BN > least && lds_bad[buf] == t + 1) {
      static_assert(BUFS * SIZE >= kAttnWaves * 1024, "room for the waves' probabilities");
      __syncthreads();  // nobody reads the keys any more: both of their buffers are free until the next keys are placed
      if (active) w.template add_nonfinite<NT>(lds_k[0] + wave * 1024, lds_v[buf], key0, s);
      __syncthreads();
      clear_nonfinite(lds_v[buf], SIZE, threadIdx.x, 256);
      __syncthreads();
    }
    if constexpr (BUFS == 1) __syncthreads();
    if (more) {
      stage.store(lds_k[other], a.D);
      fetch_v(t + 1);
    }
    if (active) w.template values<NT>(lds_v[buf], s);
    if constexpr (BUFS == 1) __syncthreads();
    if (more) place_v(t + 1, other);
    __syncthreads();
  };

  if (t_begin < t_end) {
    fetch_k(t_begin);
    stage.store(lds_k[0], a.D);
    fetch_v(t_begin);
    __syncthreads();  // lds_bad
    place_v(t_begin, 0);
    __syncthreads();
    for (int t = t_begin; t < t_end; t += BUFS) {
      work(t, Const<0>{});
      if (BUFS == 2 && t + 1 < t_end) work(t + 1, Const<BUFS - 1>{});
    }
  }

  const float l = halves_sum(w.l);
  if (w.row >= rows) return;
  const int64_t at = (seq.q_off + w.token) * a.H + w.head;
  const int64_t part = (((int64_t)id * a.KV + kvh) * a.splits + split) * kAttnRows + wave * 32 + (w.lane & 31);
  const float inv = a.splits == 1 ? inverse_sum(l) : 1.f;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = d * 32 + 8 * g + 4 * w.half;
      const float x[4] = {w.o[d][g * 4] * inv, w.o[d][g * 4 + 1] * inv, w.o[d][g * 4 + 2] * inv, w.o[d][g * 4 + 3] * inv};
      if (a.splits == 1)
        store_out<T>(a, at, col, x);
      else
        store4<float>(a.part_o + part * a.D, col, a.D, x);
    }
  if (w.half == 0) {
    if (a.splits > 1) {
      a.part_ml[part * 2] = w.m;
      a.part_ml[part * 2 + 1] = l;
    } else if (a.lse) {
      a.lse[at] = log_sum<T>(a, w.m, l);
    }
  }
}

// ---- few rows: 32 of them, the waves of a workgroup divide the keys ----------------------------------------------------
// Bound: the bytes of the keys and values.  A wave fetches its own tiles of 32 keys into its own part of LDS, so there is no
// barrier in the loop and each wave keeps a tile of keys and one of values in flight; keys and values take turns in one
// place (a wave's LDS accesses happen in order).  The waves' sums meet in LDS at the end.
// With large heads the rows stand in LDS, one tile for all waves, and only one of keys and values is on its way at a time, of
// fp32 heads past 128 only half a tile, or registers spill (135 with bf16 heads of 256, 604 with fp32 ones).  8 heads, one token,
// 16 caches of up to 8192 rows: bf16 heads of 256 605 -> 130 us (4.9 TB/s), of 192 114 -> 109 us; fp32, up to 4096 rows, of 128
// 104 -> 94 us (4.0 TB/s), of 256 670 us with whole tiles, 522 with halves, 430 with the threads' columns fixed (1.2 TB/s: bound by
// the splitting into thirds); fp32 heads of 192 on one key head, five tokens: 210 -> 77 us.  Smaller heads have the registers to
// keep both on their way.
template <typename T, int HD>
constexpr int few_waves() { return Kind<T>::P == 3 && HD > 128 ? 2 : 4; }
template <typename T, int HD>
constexpr bool few_large() { return HD > (Kind<T>::P == 1 ? 128 : 64); }

template <typename T, int HD>
__global__ __launch_bounds__((64 * few_waves<T, HD>())) void attn_few_rows_kernel(const AttnArgs a) {
  typedef typename Kind<T>::U U;
  constexpr int HDP = attn_pow2(HD);
  constexpr int W = few_waves<T, HD>();
  constexpr int SIZE = Kind<T>::P * 32 * HDP;
  constexpr int TILES = W * SIZE * (int)sizeof(U), JOIN = 32 * HD * (int)sizeof(float);
  __shared__ __attribute__((aligned(16))) char lds[TILES > JOIN ? TILES : JOIN];
  constexpr bool kLarge = few_large<T, HD>();
  __shared__ __attribute__((aligned(16))) U lds_q[kLarge ? SIZE : 8];
  __shared__ U lds_p[W][32 * 32];
  __shared__ float lds_ml[W][32][2];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const int split = (int)(id % a.splits);
  id /= a.splits;
  const AttnSeq seq = locate_rows<32>(a, id);
  if (!seq.found) {
    if (a.capacity == 0 && split == 0) clear_behind<T, 32>(a, seq, kvh);
    return;
  }
  const int rows = seq.q_len * a.G;
  const int row0 = seq.tile * 32;
  if (row0 >= rows) return;
  AttnWave<T, HD, (Kind<T>::P == 3 && HD > 192)> w;
  w.begin(a, seq, kvh, row0, rows, !kLarge);
  if constexpr (kLarge) {
    TileStage<T, HD, 32, 64 * W> stage;
    const int token0 = div_g(a, row0);
    stage.fetch_rows(static_cast<const T*>(a.q) + (seq.q_off + token0) * a.q_row + (int64_t)kvh * a.G * a.q_head, [&](int i) {
      const int row = min(row0 + i, rows - 1), token = div_g(a, row);
      return (token - token0) * (int)a.q_row + (row - token * a.G) * (int)a.q_head;
    }, a.D, rows - row0);
    stage.store(lds_q, a.D);
    __syncthreads();
  }
  const int tiles = (w.most + 31) / 32;
  const int per_split = (tiles + a.splits - 1) / a.splits;
  const int t_end = min(tiles, (split + 1) * per_split);
  const T* k = static_cast<const T*>(a.k) + seq.b * a.k_batch + seq.s_off * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + seq.b * a.v_batch + seq.s_off * a.v_row + (int64_t)kvh * a.v_head;
  U* tile = reinterpret_cast<U*>(lds) + wave * SIZE;

  constexpr bool kHalf = Kind<T>::P == 3 && HD > 128;
  constexpr int SR = kHalf ? 16 : 32;
  TileStage<T, HD, SR, 64, 32> stage_k, stage_own;
  auto& stage_v = [&]() -> TileStage<T, HD, SR, 64, 32>& {
    if constexpr (kLarge) return stage_k;
    else return stage_own;
  }();
  auto fetch_k = [&](int t, int r = 0) { stage_k.fetch(k + (int64_t)(t * 32 + r) * a.k_row, a.k_row, a.D, seq.s_len - t * 32 - r); };
  auto fetch_v = [&](int t, int r = 0) { stage_v.fetch(v + (int64_t)(t * 32 + r) * a.v_row, a.v_row, a.D, seq.s_len - t * 32 - r); };
  int t = __builtin_amdgcn_readfirstlane(split * per_split + wave);
  if (t < t_end) {
    fetch_k(t);
    if (!kLarge) fetch_v(t);
  }
  for (; t < t_end; t += W) {
    const int key0 = t * 32;
    f32x16 s[1];
    wave_order();
    stage_k.store(tile, a.D);
    if constexpr (kHalf) {
      fetch_k(t, 16);
      stage_k.store(tile + 16 * HDP, a.D);
    }
    if (kLarge)
      fetch_v(t);
    else if (t + W < t_end)
      fetch_k(t + W);
    wave_order();
    w.template scores<1, kLarge>(tile, lds_q, key0, s);
    wave_order();
    stage_v.store(tile, a.D);
    bool first = false;  // of a tile that comes in halves
    if constexpr (kHalf) {
      first = key0 + 32 > w.least && stage_v.nonfinite();
      fetch_v(t, 16);
      stage_v.store(tile + 16 * HDP, a.D);
    }
    wave_order();
    if (key0 + 32 > w.least && __any(first || stage_v.nonfinite())) {
      w.template add_nonfinite<1>(lds_p[wave], tile, key0, s);
      wave_order();
      clear_nonfinite(tile, SIZE, threadIdx.x & 63, 64);
      wave_order();
    }
    if (t + W < t_end) {
      if (kLarge)
        fetch_k(t + W);
      else
        fetch_v(t + W);
    }
    w.template values<1>(tile, s);
  }

  // the waves' parts: maximum, sums, then the rows one wave after another (a fixed order)
  {
    const float l = halves_sum(w.l);
    if (w.half == 0) {
      lds_ml[wave][w.lane][0] = w.m;
      lds_ml[wave][w.lane][1] = l;
    }
  }
  __syncthreads();
  float m = -__builtin_inff(), l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, lds_ml[i][w.lane & 31][0]);
#pragma unroll
  for (int i = 0; i < W; ++i) l = fmaf(lds_ml[i][w.lane & 31][1], prob_weight<T>(lds_ml[i][w.lane & 31][0], m, w.c2), l);
  const float f = prob_weight<T>(w.m, m, w.c2) * (a.splits == 1 ? inverse_sum(l) : 1.f);
  float* join = reinterpret_cast<float*>(lds);
  auto join_at = [](int r, int col) { return r * HD + (((col >> 2) ^ (r & 7)) << 2); };  // 8 rows at one column: 8 places
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (wave == i) {
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4v* to = reinterpret_cast<f32x4v*>(join + join_at(w.lane & 31, d * 32 + 8 * g + 4 * w.half));
          f32x4v x = {w.o[d][g * 4] * f, w.o[d][g * 4 + 1] * f, w.o[d][g * 4 + 2] * f, w.o[d][g * 4 + 3] * f};
          if (i > 0) x += *to;
          *to = x;
        }
    }
    __syncthreads();
  }
  const int64_t part = (((int64_t)id * a.KV + kvh) * a.splits + split) * 32;
  if (wave == 0 && w.half == 0 && w.row < rows) {
    if (a.splits > 1) {
      a.part_ml[(part + w.lane) * 2] = m;
      a.part_ml[(part + w.lane) * 2 + 1] = l;
    } else if (a.lse) {
      a.lse[(seq.q_off + w.token) * a.H + w.head] = log_sum<T>(a, m, l);
    }
  }
  for (int i = threadIdx.x; i < 32 * (HD / 4); i += 64 * W) {
    const int r = i / (HD / 4), col = i % (HD / 4) * 4;
    if (row0 + r >= rows) break;
    const f32x4v y = *reinterpret_cast<const f32x4v*>(join + join_at(r, col));
    const float x[4] = {y[0], y[1], y[2], y[3]};
    const int token = div_g(a, row0 + r);
    if (a.splits == 1)
      store_out<T>(a, (seq.q_off + token) * a.H + (int64_t)kvh * a.G + (row0 + r - token * a.G), col, x);
    else
      store4<float>(a.part_o + (part + r) * a.D, col, a.D, x);
  }
}

// Joins the parts of a row tile's keys: one wave per row, first its lanes over the parts (at most 64), then over the columns.
template <typename T, int TILE>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int GROUPS = TILE / 4;  // workgroups of 4 rows per tile
  int64_t id = blockIdx.x;
  const int at = (int)(id % GROUPS) * 4 + wave;
  id /= GROUPS;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const AttnSeq seq = locate_rows<TILE>(a, id);
  if (!seq.found) return;
  const int row = seq.tile * TILE + at;
  if (row >= seq.q_len * a.G) return;
  const int64_t part = (((int64_t)id * a.KV + kvh) * a.splits) * TILE + at;
  const bool mine = lane < a.splits;
  const float m_part = mine ? a.part_ml[(part + (int64_t)lane * TILE) * 2] : -__builtin_inff();
  const float l_part = mine ? a.part_ml[(part + (int64_t)lane * TILE) * 2 + 1] : 0.f;
  float m = m_part;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  const float f = prob_weight<T>(m_part, m, a.scale * kLog2e);
  const float l = lanes_sum<64>(l_part * f);
  __shared__ float factor[4][64];
  factor[wave][lane] = f;
  wave_order();
  const float inv = inverse_sum(l);
  const int64_t out = [&] {
    const int token = div_g(a, row);
    return (seq.q_off + token) * a.H + (int64_t)kvh * a.G + (row - token * a.G);
  }();
  // as many lanes as the columns need (4 each), the others take other parts
  const int width = a.D <= 64 ? 16 : (a.D <= 128 ? 32 : 64);
  const int col = lane % width * 4;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = lane / width; s < a.splits; s += 64 / width) {
    const float fs = factor[wave][s];
    const float* p = a.part_o + (part + (int64_t)s * TILE) * a.D;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf(col + j < a.D ? p[col + j] : 0.f, fs, o[j]);
  }
#pragma unroll
  for (int d = 32; d >= 16; d >>= 1)
    if (d >= width) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], d, 64);
    }
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] *= inv;
  if (lane < width) store_out<T>(a, out, col, o);
  if (a.lse && lane == 0) a.lse[out] = log_sum<T>(a, m, l);
}

// The table of a pack of many sequences, by one workgroup: 1024 sequences at a time, the rows before each, then (of what is left
// of them within the totals) the tiles.
__global__ __launch_bounds__(1024) void attn_table_kernel(const AttnArgs a, int64_t* table, int row_tile, int key_tile) {
  __shared__ int64_t sums[2][2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = a.B + 1;
  int64_t before[4] = {0, 0, 0, 0};  // the workgroup's sequences
  // x, y -> what all threads before this one have of them; adds everybody's to the workgroup's
  auto scan = [&](int64_t& x, int64_t& y, int which) {
    const int64_t ix = lanes_prefix(x, lane), iy = lanes_prefix(y, lane);
    if (lane == 63) {
      sums[which][0][wave] = ix;
      sums[which][1][wave] = iy;
    }
    __syncthreads();
    x = before[2 * which] + ix - x;
    y = before[2 * which + 1] + iy - y;
#pragma unroll 1
    for (int w = 0; w < 16; ++w) {
      if (w < wave) {
        x += sums[which][0][w];
        y += sums[which][1][w];
      }
      before[2 * which] += sums[which][0][w];
      before[2 * which + 1] += sums[which][1][w];
    }
  };
  for (int i0 = 0; i0 < a.B; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    int64_t q_len = i < a.B ? clamp64(a.q_lengths[i], a.total_q) : 0, s_len = i < a.B ? clamp64(a.s_lengths[i], a.total_s) : 0;
    int64_t q = q_len, s = s_len;
    scan(q, s, 0);
    q = clamp64(q, a.total_q);
    s = clamp64(s, a.total_s);
    q_len = clamp64(q_len, a.total_q - q);
    s_len = clamp64(s_len, a.total_s - s);
    int64_t row_tiles = (q_len * a.G + row_tile - 1) / row_tile, key_tiles = key_tile > 0 ? (s_len + key_tile - 1) / key_tile : 0;
    scan(row_tiles, key_tiles, 1);
    if (i < a.B) {
      table[i] = q;
      table[n + i] = s;
      table[2 * n + i] = row_tiles;
      if (key_tile > 0) table[3 * n + i] = key_tiles;
    }
  }  // (a scan's sums are written again only behind the other scan's barrier)
  if (threadIdx.x == 0) {
    table[a.B] = clamp64(before[0], a.total_q);
    table[n + a.B] = clamp64(before[1], a.total_s);
    table[2 * n + a.B] = before[2];
    if (key_tile > 0) table[3 * n + a.B] = before[3];
  }
}

int attn_table_launch(AttnArgs& a, void* table, int row_tile, int key_tile, hipStream_t stream, const char* what) {
  if (a.B <= kAttnWalk) return 0;
  a.table = static_cast<int64_t*>(table);
  hipLaunchKernelGGL(attn_table_kernel, dim3(1), dim3(1024), 0, stream, a, static_cast<int64_t*>(table), row_tile, key_tile);
  return launch_status(what);
}

// ---- launches ----------------------------------------------------------------------------------------------------------
struct AttnPlan {
  bool few;         // 32-row tiles whose waves divide the keys, else 128-row tiles
  int64_t tiles;    // row tiles (a bound in a pack)
  int splits;
  size_t table;     // workspace: the table of the sequences, ...
  size_t bytes;     // ... and with the parts behind it
  int tile() const { return few ? 32 : kAttnRows; }
};

// `tokens` > 0: a cache, every sequence has that many queries; else a pack, whose lengths are known on the device only.
inline AttnPlan attn_plan(int B, int64_t total_q, int64_t total_s, int tokens, int KV, int G, int D) {
  AttnPlan p;
  // 32-row tiles where sequences have no more rows than that (a cache's newest tokens), and where 128-row tiles would keep
  // at most a quarter of the 256 CUs.  32-row against 128-row tiles: one sequence of 1000 tokens, 4 heads of 64: bf16 15 / 23 us,
  // fp32 29 / 64; 4 x 500 tokens, 4 heads of 256: 32 / 61, 178 / 246; at the border itself (one sequence of 2048 tokens, 4 heads
  // of 64) 22 / 25 and 50 / 46, with twice the tiles (2 x 1024 tokens, 2 key heads of 128, bf16) 40 / 37: keys and values are then
  // read by four times as many workgroups.  (Against thousands of keys, which 128-row tiles divide more often, the rule costs:
  // 2 x 500 tokens, 4000 keys, 4 heads of 64: bf16 39 / 26, fp32 94 / 48.)
  p.few = total_q * G <= (int64_t)32 * B || ceil_div(total_q * G, kAttnRows) * KV <= 64;
  p.tiles = tokens > 0 ? B * ceil_div((int64_t)tokens * G, p.tile()) : ceil_div(total_q * G, p.tile()) + B;
  // Keys are divided where the row tiles leave compute units idle, as far as every part of a sequence of the mean length
  // keeps 512 keys: into one workgroup a CU of the 32-row kernel, which is bound by memory (6 caches of 32768 rows, 4 tokens:
  // 42 us; 512 workgroups, whose parts are twice the bytes to join: 49 us), into two of the other.
  const int64_t groups = std::max<int64_t>(p.tiles * KV, 1), mean = tokens > 0 ? total_s : total_s / std::max(B, 1);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(p.few ? 256 : 512) / groups, mean / 512, 64}));
  p.table = tokens > 0 ? 0 : attn_table_bytes(B, 3);
  p.bytes = p.table + (p.splits > 1 ? (size_t)(groups * p.splits * p.tile()) * (size_t)(D + 2) * sizeof(float) : 0);
  return p;
}

template <typename T, int HD>
int attn_forward_launch(const AttnArgs& a, const AttnPlan& p, hipStream_t stream, const char* what) {
  const dim3 grid((unsigned)(p.tiles * a.KV * a.splits));
  if (p.few)
    hipLaunchKernelGGL((attn_few_rows_kernel<T, HD>), grid, dim3((64 * few_waves<T, HD>())), 0, stream, a);
  else
    hipLaunchKernelGGL((attn_forward_kernel<T, HD>), grid, dim3(256), 0, stream, a);
  int rc = launch_status(what);
  if (rc == 0 && a.splits > 1) {
    const dim3 join((unsigned)(p.tiles * a.KV * (p.tile() / 4)));
    if (p.few)
      hipLaunchKernelGGL((attn_join_kernel<T, 32>), join, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((attn_join_kernel<T, kAttnRows>), join, dim3(256), 0, stream, a);
    rc = launch_status(what);
  }
  return rc;
}

template <typename T>
int attn_forward_type(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream, const char* what) {
  switch (attn_head_size(a.D)) {
    case 32: return attn_forward_launch<T, 32>(a, plan, stream, what);
    case 64: return attn_forward_launch<T, 64>(a, plan, stream, what);
    case 96: return attn_forward_launch<T, 96>(a, plan, stream, what);
    case 128: return attn_forward_launch<T, 128>(a, plan, stream, what);
    case 192: return attn_forward_launch<T, 192>(a, plan, stream, what);
    default: return attn_forward_launch<T, 256>(a, plan, stream, what);
  }
}

int attn_check(const char* what, int dtype, int B, int64_t total_q, int64_t total_s, int H, int KV, int D,
               float scale) {
  V3D_REQUIRE(dtype == V3D_F32 || dtype == V3D_F16 || dtype == V3D_BF16, what, "unknown element type");
  V3D_REQUIRE(B >= 0 && total_q >= 0 && total_s >= 0 && H >= 1 && KV >= 1 && D >= 1, what, "bad shape");
  V3D_REQUIRE(H % KV == 0, what, "the query heads must be a multiple of the key heads");
  V3D_REQUIRE(D >= (dtype == V3D_F32 ? 4 : 8), what, "a head has at least 16 bytes");
  V3D_REQUIRE(scale > 0.f && scale < __builtin_inff(), what, "the scale must be positive and finite");
  if (D > V3D_ATTENTION_MAX_HEAD_SIZE) {
    set_last_error("%s: head size %d, at most %d", what, D, V3D_ATTENTION_MAX_HEAD_SIZE);
    return V3D_ERR_SIZE_LIMIT;
  }
  const int64_t most = (int64_t)1 << 30;
  if (total_q > most / H || total_s > most || B > (1 << 24)) {
    set_last_error("%s: more than 2^30 rows (query rows count once per head)", what);
    return V3D_ERR_SIZE_LIMIT;
  }
  return 0;
}

// A tile's rows are addressed by 32-bit byte offsets from the tile's first row: at most 128 rows of a key tensor, at most
// 129 tokens and the heads of a group of a query tensor.  (One new token a sequence of a cache: its row stride leads from
// sequence to sequence only, which is 64-bit.)
int attn_check_strides(const char* what, const AttnArgs& a) {
  const int64_t reach = (int64_t)1 << 29;  // elements of 4 bytes
  auto fits = [&](int64_t row, int64_t head) {
    return row >= 0 && head >= 0 && row < reach && head < reach && 129 * row + a.G * head + a.D < reach;
  };
  const bool alone = a.capacity > 0 && a.tokens == 1;
  if (a.q_row < 0 || !fits(alone ? 0 : a.q_row, a.q_head) || !fits(a.k_row, 0) || !fits(a.v_row, 0) || !fits((int64_t)a.H * a.D, a.D)) {
    set_last_error("%s: strides of a query or key row beyond 32-bit tile offsets", what);
    return V3D_ERR_SIZE_LIMIT;
  }
  V3D_REQUIRE((a.k_row == 0 || a.k_row >= a.D) && (a.v_row == 0 || a.v_row >= a.D), what, "key rows overlap");
  V3D_REQUIRE(a.k_head >= 0 && a.v_head >= 0 && a.k_batch >= 0 && a.v_batch >= 0, what, "negative stride");
  return 0;
}

int attn_forward_run(AttnArgs& a, int dtype, const AttnPlan& plan, void* workspace, size_t workspace_bytes, int device,
                     void* stream, const char* what) {
  const int bad = attn_check_strides(what, a);
  if (bad != 0) return bad;
  if (plan.tiles * a.KV * plan.splits > kAttnMaxGroups ||
      (plan.splits > 1 && plan.tiles * a.KV * (plan.tile() / 4) > kAttnMaxGroups)) {
    set_last_error("%s: more than 2^24 row tiles (every sequence counts as one at least, once per key head)", what);
    return V3D_ERR_SIZE_LIMIT;
  }
  DeviceGuard guard(device);
  if (guard.rc != 0) return guard.rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  a.splits = plan.splits;
  Scratch ws;
  if (plan.bytes > 0) {
    const int rc = ws.acquire(what, workspace, workspace_bytes, plan.bytes, s);
    if (rc != 0) return rc;
    a.part_o = reinterpret_cast<float*>(ws.base + plan.table);
    a.part_ml = a.part_o + plan.tiles * a.KV * a.splits * plan.tile() * a.D;
  }
  int rc = plan.table > 0 ? attn_table_launch(a, ws.base, plan.tile(), 0, s, what) : 0;
  if (rc == 0)
    rc = dtype == V3D_F32   ? attn_forward_type<float>(a, plan, s, what)
         : dtype == V3D_F16 ? attn_forward_type<f16>(a, plan, s, what)
                            : attn_forward_type<bf16>(a, plan, s, what);
  return ws.release(what, rc);
}

}  // namespace v3d

extern "C" {

size_t v3d_attention_pack_workspace_bytes(int B, int64_t total_q, int64_t total_s, int H, int KV, int D) {
  if (B < 0 || total_q <= 0 || total_s < 0 || H <= 0 || KV <= 0 || H % KV != 0 || D <= 0) return 0;
  return v3d::attn_plan(B, total_q, total_s, 0, KV, H / KV, D).bytes;
}

int v3d_attention_pack_plan(int dtype, int B, int64_t total_q, int64_t total_s, int H, int KV, int D, int* row_tile,
                            int* key_parts, int* grad_key_parts, int* grad_row_parts) {
  using namespace v3d;
  const int rc = attn_check("attention_pack_plan", dtype, B, total_q, total_s, H, KV, D, 1.f);
  if (rc != 0) return rc;
  const AttnPlan plan = attn_plan(B, total_q, total_s, 0, KV, H / KV, D);
  if (row_tile != nullptr) *row_tile = plan.tile();
  if (key_parts != nullptr) *key_parts = plan.splits;
  if (grad_key_parts != nullptr) *grad_key_parts = attn_backward_q_splits(dtype, B, total_q, total_s, KV, H / KV);
  if (grad_row_parts != nullptr) *grad_row_parts = attn_backward_splits(B, total_s, KV, D);
  return 0;
}

int v3d_attention_pack_fwd(const void* q, const void* k, const void* v, const int64_t* q_lengths,
                           const int64_t* s_lengths, void* out, void* rest, float* lse, int dtype, int B,
                           int64_t total_q, int64_t total_s, int H, int KV, int D, const int64_t* strides, float scale,
                           int causal,
                           void* workspace, size_t workspace_bytes, int device, void* stream) {
  using namespace v3d;
  const char* what = "attention_pack";
  int rc = attn_check(what, dtype, B, total_q, total_s, H, KV, D, scale);
  if (rc != 0) return rc;
  if (total_q == 0) return 0;
  V3D_REQUIRE(q && out && strides && (B == 0 || (q_lengths && s_lengths)) && (total_s == 0 || (k && v)), what,
              "null pointer");
  AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.rest = dtype == V3D_F32 ? nullptr : rest;
  a.lse = lse;
  a.q_lengths = q_lengths;
  a.s_lengths = s_lengths;
  a.total_q = total_q;
  a.total_s = total_s;
  a.q_row = strides[0];
  a.q_head = strides[1];
  a.k_row = strides[2];
  a.k_head = strides[3];
  a.v_row = strides[4];
  a.v_head = strides[5];
  a.B = B;
  attn_heads(a, H, KV, D);
  a.scale = scale;
  a.causal = causal;
  return attn_forward_run(a, dtype, attn_plan(B, total_q, total_s, 0, KV, a.G, D), workspace, workspace_bytes, device,
                          stream, what);
}

size_t v3d_cached_attention_workspace_bytes(int B, int tokens, int64_t capacity, int H, int KV, int D) {
  if (B <= 0 || tokens <= 0 || H <= 0 || KV <= 0 || H % KV != 0 || D <= 0) return 0;
  return v3d::attn_plan(B, (int64_t)B * tokens, capacity, tokens, KV, H / KV, D).bytes;
}

int v3d_cached_attention(const void* q, const void* k_cache, const void* v_cache, const int64_t* lengths, void* out,
                         int dtype, int B, int tokens, int64_t capacity, int H, int KV, int D, const int64_t* strides,
                         float scale, void* workspace, size_t workspace_bytes, int device, void* stream) {
  using namespace v3d;
  const char* what = "cached_attention";
  V3D_REQUIRE(B >= 0 && tokens >= 0 && capacity >= 1, what, "bad shape");
  int rc = attn_check(what, dtype, B, (int64_t)B * tokens, capacity, H, KV, D, scale);
  if (rc != 0) return rc;
  if (B == 0 || tokens == 0) return 0;
  V3D_REQUIRE(q && k_cache && v_cache && lengths && out && strides, what, "null pointer");
  AttnArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.s_lengths = lengths;
  a.total_q = (int64_t)B * tokens;
  a.total_s = capacity;
  a.q_row = strides[0];
  a.q_head = strides[1];
  a.k_batch = strides[2];
  a.k_row = strides[3];
  a.k_head = strides[4];
  a.v_batch = strides[5];
  a.v_row = strides[6];
  a.v_head = strides[7];
  a.capacity = capacity;
  a.tokens = tokens;
  a.B = B;
  attn_heads(a, H, KV, D);
  a.scale = scale;
  a.causal = 1;
  return attn_forward_run(a, dtype, attn_plan(B, a.total_q, capacity, tokens, KV, a.G, D), workspace, workspace_bytes,
                          device, stream, what);
}

}  // extern "C"
