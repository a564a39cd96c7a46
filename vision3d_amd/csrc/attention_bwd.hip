// attention_bwd.hip -- the gradients of attention_pack.
//
//   p_ij = exp(s_ij - lse_i),  dv_j = sum_i p_ij do_i,  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// Two kernels, each the owner of what it writes, so there are no atomics and the same input gives the same bits: one goes
// over the keys of a row tile (dq, and delta on the way), one over the rows of a key tile (dk, dv; the rows of all G query
// heads of a key head are folded, so the sum over a group needs nothing extra).  Both form s and dp again: 7 products
// instead of the 5 that the sums need, where a single kernel would add dq with atomics in fp32.  Where tiles leave compute units
// idle, the keys of a row tile and the rows of a key tile are divided and their sums joined in a fixed order.
//
// Measured, 8 x 2048 tokens, 16/4 heads of 128, bf16, no mask: dq 449 us = 918 TFLOP/s (two waves a SIMD), dk / dv 869 us = 633
// TFLOP/s (one wave: its products and exponentials take turns).  8192 causal tokens in 5 sequences: dq 130 us, dk / dv 260 us
// and 18 us to join its parts.
#include <algorithm>

#include "attn.h"

namespace v3d {

struct AttnBwdArgs {
  AttnArgs f;          // q, k, v, out, lse and the geometry of the forward (never a cache)
  const void* grad;    // (total_q, H, D) contiguous
  float* delta;        // (total_q, H): written by the dq kernel, read by the dk / dv kernel
  int q_splits;        // parts that the keys of a row tile are divided into
  float* part_q;       // q_splits > 1: (q_splits, total_q, H, D) sums of the parts
  int splits;          // parts that the rows of a key tile are divided into
  float* part;         // splits > 1: (splits, 2, total_s, KV, D) sums of the parts, dk's and dv's
  float* grad_norm;    // fp16: (total_q, H) 2-norms of the rows of grad, written by the dq kernel ...
  float* value_norm;   // ... and (total_s, KV) of the values, written before it; infinities and NaN count as 0
  void* dq;            // (total_q, H, D) or NULL, (total_s, KV, D), contiguous
  void* dk;
  void* dv;
};

// ---- the range of fp16 -------------------------------------------------------------------------------------------------
// fp16 holds 11 bits down to 2^-14 and nothing below 2^-25 or above 2^16, and p, about 1 / keys, and ds, about grad . v / keys,
// leave that range long before the gradients do (4096 keys, gradients of 1e-3: 5e-3 off, of 1e-4: 5e-2).  So both meet their
// product times a power of two, which the 32-bit sums are divided by at the end: p times 2^kLift, in the exponent; ds times a
// factor of its row (dq) or key (dk) that puts a bound of it at 2^11 ... 2^12:
//   |ds_ij| <= p_ij (|do_i . v_j| + |do_i . o_i|) <= 2 |do_i| max |v_j|,
// with the 2-norms, the largest taken over the sequence (a factor that follows the largest ds would have to rescale the sums:
// the registers of heads of 256 spill).  A typical ds of 2000 keys then lies at 2^-2, what is 2^-37 of the bound is still held,
// and a p that 32-bit scores put past 1 has room.  Costs 2 to 6 % of a training step (8192 causal tokens in 5 sequences, 16/4
// heads of 128: 464 -> 484 us; 8 x 2048 tokens without a mask 2030 -> 2070 us, 8 us of it the values' norms).
template <typename T>
constexpr bool kFp16 = __is_same(T, f16);
template <typename T>
constexpr float kLift = kFp16<T> ? 12.f : 0.f;

__device__ __forceinline__ float range_exponent(float bound) {  // e: bound * 2^e in [2^11, 2^12), within what factors can undo
  return (float)min(max(11 + 127 - (int)(__float_as_uint(bound) >> 23), -60), 60);
}
__device__ __forceinline__ float finite_norm(float squares) {
  const float n = sqrtf(squares);
  return n < __builtin_inff() ? n : 0.f;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
  return x;
}

// 16 lanes a row; a workgroup stays with one key head.
__global__ __launch_bounds__(256) void attn_value_norm_kernel(const AttnBwdArgs b) {
  const AttnArgs& a = b.f;
  const unsigned kvh = blockIdx.x % (unsigned)a.KV, group = blockIdx.x / (unsigned)a.KV, groups = gridDim.x / (unsigned)a.KV;
  for (int64_t row = group * 16 + threadIdx.x / 16; row < a.total_s; row += groups * 16) {
    const f16* v = static_cast<const f16*>(a.v) + row * a.v_row + kvh * a.v_head;
    float sum = 0.f;
    for (int c = (threadIdx.x & 15) * 8; c < a.D; c += 128) {
      float x[8];
      if (c + 8 <= a.D) {
        load_vec<f16, 8>(v + c, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < a.D ? to_f32(v[c + j]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
    }
    sum = lanes_sum<16>(sum);
    if ((threadIdx.x & 15) == 0) b.value_norm[row * a.KV + kvh] = finite_norm(sum);
  }
}

// Keys (or rows) of a tile that passes by; two of them (fp32 heads past 128: one), of two tensors, in LDS.
template <typename T, int HD>
constexpr int bwd_tile() { return Kind<T>::P == 1 && HD <= 64 ? 64 : 32; }
template <typename T, int HD>
constexpr int bwd_buffers() { return Kind<T>::P == 3 && HD > 128 ? 1 : 2; }

// Tiles [0, count) pass by: `fetch` starts the loads of one into registers, `place` puts them into LDS, `work` uses it.  With
// two buffers a tile is fetched two tiles ahead of its use (a tile's work is shorter than a load's way from memory); loads
// past the last tile read nothing but are issued all the same, so that waiting for the older ones stays countable.
template <int BUFS, typename Fetch, typename Place, typename Work>
__device__ __forceinline__ void pass_tiles(int count, Fetch fetch, Place place, Work work) {
  if (count <= 0) return;
  if constexpr (BUFS == 2) {
    fetch(0, Const<0>{});
    fetch(1, Const<1>{});
    place(Const<0>{});
    __syncthreads();
    for (int t = 0; t < count; t += 2) {
      fetch(t + 2, Const<0>{});
      work(t, Const<0>{});
      place(Const<1>{});
      __syncthreads();
      if (t + 1 >= count) break;
      fetch(t + 3, Const<1>{});
      work(t + 1, Const<1>{});
      place(Const<0>{});
      __syncthreads();
    }
  } else {
    fetch(0, Const<0>{});
    place(Const<0>{});
    __syncthreads();
    for (int t = 0; t < count; ++t) {
      fetch(t + 1, Const<0>{});
      work(t, Const<0>{});
      __syncthreads();
      place(Const<0>{});
      __syncthreads();
    }
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(256, HD <= (Kind<T>::P == 1 ? 128 : 64) ? 2 : 1) void attn_backward_q_kernel(const AttnBwdArgs b) {
  constexpr int HDP = attn_pow2(HD);
  constexpr int BN = bwd_tile<T, HD>();
  constexpr int NT = BN / 32;
  constexpr int BUFS = bwd_buffers<T, HD>();
  constexpr int STEPS = HD / 16;
  constexpr bool kAgain = Kind<T>::P == 3 && HD > 192;  // see again()
  constexpr int DT = HD / 32;
  typedef typename Kind<T>::U U;
  __shared__ __attribute__((aligned(16))) U lds_k[BUFS][Kind<T>::P * BN * HDP];
  __shared__ __attribute__((aligned(16))) U lds_v[BUFS][Kind<T>::P * BN * HDP];

  const AttnArgs& a = b.f;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const int split = (int)(id % b.q_splits);
  const AttnSeq seq = locate_rows<kAttnRows>(a, id / b.q_splits);
  T* dq = static_cast<T*>(b.dq);
  float* pq = b.part_q + split * (a.total_q * a.H * a.D);
  if (!seq.found) {  // rows behind the last sequence have no gradient
    if (dq == nullptr) return;
    const int64_t rows = (a.total_q - seq.q_end) * a.G;
    for (int i = threadIdx.x; i < kAttnRows; i += 256) {
      const int64_t r = seq.spare * kAttnRows + i;
      if (r >= rows) break;
      const int64_t at = (seq.q_end + r / a.G) * a.H + (int64_t)kvh * a.G + r % a.G;
      for (int64_t d = at * a.D; d < (at + 1) * a.D; ++d) {
        if (b.q_splits == 1)
          dq[d] = (T)0.f;
        else
          pq[d] = 0.f;
      }
    }
    return;
  }
  const int rows = seq.q_len * a.G;
  const int row0 = seq.tile * kAttnRows;
  if (row0 >= rows) return;  // lengths that overrun the total were cut
  const int row = row0 + wave * 32 + (lane & 31);
  const int token = div_g(a, min(row, rows - 1));
  const int head = kvh * a.G + min(row, rows - 1) - token * a.G;
  const int limit = attn_limit(a, seq, token);
  const int wave_least = __builtin_amdgcn_readfirstlane(limit);
  const int wave_most =
      row0 + wave * 32 < rows ? attn_limit(a, seq, div_g(a, min(row0 + wave * 32 + 31, rows - 1))) : 0;
  const int most = attn_limit(a, seq, div_g(a, min(row0 + kAttnRows - 1, rows - 1)));
  const int tiles = (most + BN - 1) / BN, per_split = (tiles + b.q_splits - 1) / b.q_splits;
  const int t_begin = split * per_split, t_end = min(tiles, t_begin + per_split);

  const int token0 = div_g(a, row0);
  const T* q = static_cast<const T*>(a.q) + (seq.q_off + token0) * a.q_row + (int64_t)kvh * a.G * a.q_head;
  const T* k = static_cast<const T*>(a.k) + seq.s_off * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + seq.s_off * a.v_row + (int64_t)kvh * a.v_head;
  const int64_t at = (seq.q_off + token) * a.H + head;
  const int64_t at0 = ((seq.q_off + token0) * a.H + (int64_t)kvh * a.G) * a.D;
  const int at_row = (int)(at * a.D - at0);

  TileStage<T, HD, BN, 256> stage_k[BUFS], stage_v[BUFS];
  auto fetch = [&](int t, auto to) {
    const int key0 = (t_begin + t) * BN;
    stage_k[decltype(to)::value].fetch(k + (int64_t)key0 * a.k_row, a.k_row, a.D, seq.s_len - key0);
    stage_v[decltype(to)::value].fetch(v + (int64_t)key0 * a.v_row, a.v_row, a.D, seq.s_len - key0);
  };
  auto place_tile = [&](auto from) {
    stage_k[decltype(from)::value].store(lds_k[decltype(from)::value], a.D);
    stage_v[decltype(from)::value].store(lds_v[decltype(from)::value], a.D);
  };

  Held<T, HD> qf, gf;
  float delta = 0.f;
  qf.load(q, (token - token0) * (int)a.q_row + (head - kvh * a.G) * (int)a.q_head, half, a.D, true);
  gf.load(static_cast<const T*>(b.grad) + at0, at_row, half, a.D, true);
  // delta = grad . out, the output as it was before it was rounded
  auto add_delta = [&](const void* out) {
    Held<T, HD> of;
    of.load(static_cast<const T*>(out) + at0, at_row, half, a.D, true);
    gf.begin();
    of.begin();
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const Op<T> gs = gf.get(st), os = of.get(st);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(number(gs, j), number(os, j), delta);
    }
  };
  add_delta(a.out);
  if (a.rest != nullptr) add_delta(a.rest);
  delta = halves_sum(delta);
  float lse = a.lse[at];
  if (split == 0 && half == 0 && row < rows) b.delta[at] = delta;
  float range = 0.f;  // log2 of what ds is multiplied by: in the exponent, no instruction more
  if constexpr (kFp16<T>) {
    float squares = 0.f, most_v = 0.f;
    gf.begin();
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const Op<T> gs = gf.get(st);
#pragma unroll
      for (int j = 0; j < 8; ++j) squares = fmaf(number(gs, j), number(gs, j), squares);
    }
    const float norm = finite_norm(halves_sum(squares));
    if (split == 0 && half == 0 && row < rows) b.grad_norm[at] = norm;
    if (dq == nullptr) return;
#pragma unroll 8
    for (int j = threadIdx.x; j < most; j += 256)
      most_v = fmaxf(most_v, b.value_norm[(seq.s_off + j) * a.KV + kvh]);
    __shared__ float lds_norm[4];
    most_v = wave_max(most_v);
    if (lane == 0) lds_norm[wave] = most_v;
    __syncthreads();
    most_v = fmaxf(fmaxf(lds_norm[0], lds_norm[1]), fmaxf(lds_norm[2], lds_norm[3]));
    range = range_exponent(2.f * norm * most_v);
    lse -= range;
  }

  if (dq == nullptr) return;  // only what the other kernel needs

  const float c2 = a.scale * kLog2e;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = zero16();

  auto work = [&](int t, auto buffer) {
    constexpr int buf = decltype(buffer)::value;
    const int key0 = (t_begin + t) * BN;
    if (key0 >= wave_most) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x16 s = zero16(), dp = zero16();
      qf.begin();
      gf.begin();
      const int cols = again<kAgain>(lane) & 31;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        s = product<T>(read_cols<T, HDP, BN>(lds_k[buf], n * 32 + cols, st, half), qf.get(st), s);
        dp = product<T>(read_cols<T, HDP, BN>(lds_v[buf], n * 32 + cols, st, half), gf.get(st), dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_fast(fmaf(s[r], c2, -lse)) * (dp[r] - delta);
      if (key0 + BN > wave_least) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + n * 32 + acc_row(r, half) >= limit) s[r] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Op<T> ds = pack_rows<T>(s, u);
        const int at = again<kAgain>(lane) & 63;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          acc[d] = product<T>(read_rows<T, HDP, BN>(lds_k[buf], n * 32, u, d * 32, at), ds, acc[d]);
      }
    }
  };

  pass_tiles<BUFS>(t_end - t_begin, fetch, place_tile, work);
  if (row >= rows) return;
  if (b.q_splits == 1)
    store_rows<T, DT>(dq + at * a.D, acc, a.scale * exp2_fast(-range), a.D, half);
  else
    store_rows<float, DT>(pq + at * a.D, acc, a.scale * exp2_fast(-range), a.D, half);
}

// dk and dv of a tile of 32 GROUPS keys.  A wave keeps 32 keys: their operands and both sums, 320 registers with 16-bit heads
// of 128, one wave on a SIMD.  Where that does not fit the 512 registers two waves share 32 keys, one sums dv, the other dk,
// and both form s: 40 products instead of 32, but nothing is spilled (16-bit heads of 256: 362 registers otherwise).  Up to
// there the single wave is faster although it has a SIMD to itself: 8 x 2048 tokens, 16/4 heads of 128, bf16, no mask: 869 us
// against 932 (633 and 590 TFLOP/s of the 32 products), heads of 64: 404 us against 596.
template <typename T, int HD>
constexpr bool kv_roles() { return HD > (Kind<T>::P == 1 ? 128 : 96); }
template <typename T, int HD>
constexpr int kv_groups() { return kv_roles<T, HD>() ? 2 : 4; }
constexpr int kKvThreads = 256;

template <typename T, int HD>
__global__ __launch_bounds__(kKvThreads, HD <= 32 ? 2 : 1) void attn_backward_kv_kernel(const AttnBwdArgs b) {
  constexpr int HDP = attn_pow2(HD);
  constexpr int BM = 32;
  constexpr int NT = BM / 32;
  constexpr int BUFS = bwd_buffers<T, HD>();
  constexpr int STEPS = HD / 16;
  constexpr bool kAgain = Kind<T>::P == 3 && HD > 192;  // see again()
  constexpr int DT = HD / 32;
  constexpr int GROUPS = kv_groups<T, HD>(), KEYS = 32 * GROUPS, THREADS = kKvThreads;
  constexpr bool kRoles = kv_roles<T, HD>();
  typedef typename Kind<T>::U U;
  __shared__ __attribute__((aligned(16))) U lds_q[BUFS][Kind<T>::P * BM * HDP];
  __shared__ __attribute__((aligned(16))) U lds_g[BUFS][Kind<T>::P * BM * HDP];
  __shared__ float lds_lse[BUFS][BM], lds_delta[BUFS][BM];
  __shared__ int lds_limit[BUFS][BM];

  const AttnArgs& a = b.f;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5;
  const bool keys_role = !kRoles || wave >= GROUPS;  // this wave sums dk (without roles dv too), else dv
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const int split = (int)(id % b.splits);
  const AttnSeq seq = locate_keys<KEYS>(a, id / b.splits);
  T* dk = static_cast<T*>(b.dk);
  T* dv = static_cast<T*>(b.dv);
  const int64_t plane = a.total_s * a.KV * a.D;
  float* pk = b.part + 2 * split * plane;
  float* pv = pk + plane;
  if (!seq.found) {  // keys behind the last sequence have no gradient
    for (int i = threadIdx.x; i < KEYS; i += THREADS) {
      const int64_t r = seq.s_end + seq.spare * KEYS + i;
      if (r >= a.total_s) break;
      for (int64_t d = (r * a.KV + kvh) * a.D; d < (r * a.KV + kvh + 1) * a.D; ++d) {
        if (b.splits == 1)
          dk[d] = dv[d] = (T)0.f;
        else
          pk[d] = pv[d] = 0.f;
      }
    }
    return;
  }
  const int key0 = seq.tile * KEYS;
  if (key0 >= seq.s_len) return;  // cut
  const int wave_key = key0 + wave % GROUPS * 32;
  const int key = wave_key + (lane & 31);
  const bool live = key < seq.s_len;
  const int rows = seq.q_len * a.G;
  // rows that see a key: tokens from key - (s_len - q_len) on
  const int first = a.causal ? max(0, key0 - (seq.s_len - seq.q_len)) * a.G : 0;
  const int wave_first = a.causal ? max(0, wave_key - (seq.s_len - seq.q_len)) * a.G : 0;

  const T* k = static_cast<const T*>(a.k) + (seq.s_off + key0) * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + (seq.s_off + key0) * a.v_row + (int64_t)kvh * a.v_head;
  const T* q = static_cast<const T*>(a.q) + seq.q_off * a.q_row + (int64_t)kvh * a.G * a.q_head;
  const T* grad = static_cast<const T*>(b.grad) + (seq.q_off * a.H + (int64_t)kvh * a.G) * a.D;
  const float* lse = a.lse + seq.q_off * a.H + kvh * a.G;
  const float* delta = b.delta + seq.q_off * a.H + kvh * a.G;

  const int blocks = max(0, (rows - first / BM * BM + BM - 1) / BM), per = (blocks + b.splits - 1) / b.splits;
  const int begin = first / BM * BM + split * per * BM, end = min(rows, begin + per * BM);
  TileStage<T, HD, BM, THREADS> stage_q[BUFS], stage_g[BUFS];
  float stage_lse[BUFS], stage_delta[BUFS];
  int stage_limit[BUFS];
  auto fetch = [&](int t, auto to) {
    constexpr int st = decltype(to)::value;
    const int row0 = min(begin + t * BM, rows);
    const int tok0 = div_g(a, row0);
    stage_q[st].fetch_rows(q + tok0 * a.q_row, [&](int r) {
      const int tok = div_g(a, row0 + r);
      return (tok - tok0) * (int)a.q_row + (row0 + r - tok * a.G) * (int)a.q_head;
    }, a.D, rows - row0);
    stage_g[st].fetch_rows(grad + (int64_t)tok0 * a.H * a.D, [&](int r) {
      const int tok = div_g(a, row0 + r);
      return ((tok - tok0) * a.H + (row0 + r - tok * a.G)) * a.D;
    }, a.D, rows - row0);
    if (threadIdx.x < BM) {
      const int r = min(row0 + (int)threadIdx.x, rows - 1);
      const int tok = div_g(a, r);
      const int64_t i = (int64_t)tok * a.H + (r - tok * a.G);
      stage_lse[st] = lse[i];
      stage_delta[st] = delta[i];
      stage_limit[st] = row0 + (int)threadIdx.x < rows ? attn_limit(a, seq, tok) : 0;  // a row past the last sees no key
    }
  };
  auto place_tile = [&](auto from) {
    constexpr int buf = decltype(from)::value;
    stage_q[buf].store(lds_q[buf], a.D);
    stage_g[buf].store(lds_g[buf], a.D);
    if (threadIdx.x < BM) {
      lds_lse[buf][threadIdx.x] = stage_lse[buf] - kLift<T>;  // p below is 2^kLift times as large
      lds_delta[buf][threadIdx.x] = stage_delta[buf];
      lds_limit[buf][threadIdx.x] = stage_limit[buf];
    }
  };

  float range = 1.f;  // what ds is multiplied by
  if constexpr (kFp16<T>) {
    float most_g = 0.f;
#pragma unroll 8
    for (int r = first + threadIdx.x; r < rows; r += THREADS) {
      const int tok = div_g(a, r);
      most_g = fmaxf(most_g, b.grad_norm[(seq.q_off + tok) * a.H + kvh * a.G + (r - tok * a.G)]);
    }
    __shared__ float lds_norm[4];
    most_g = wave_max(most_g);
    if (lane == 0) lds_norm[wave] = most_g;
    __syncthreads();
    most_g = fmaxf(fmaxf(lds_norm[0], lds_norm[1]), fmaxf(lds_norm[2], lds_norm[3]));
    const float norm = live ? b.value_norm[(seq.s_off + key) * a.KV + kvh] : 0.f;
    range = exp2_fast(range_exponent(2.f * most_g * norm) - kLift<T>);  // p brings its own factor
  }

  Held<T, HD> kf, vf;
  kf.load(k, (key - key0) * (int)a.k_row, half, a.D, live);
  vf.load(v, (key - key0) * (int)a.v_row, half, a.D, live);
  const float c2 = a.scale * kLog2e;
  f32x16 acc[DT], other[kRoles ? 1 : DT];  // of the wave's role, or dk and dv
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = zero16();
#pragma unroll
  for (int d = 0; d < (kRoles ? 1 : DT); ++d) other[d] = zero16();

  auto work = [&](int t, auto buffer) {
    constexpr int buf = decltype(buffer)::value;
    const int row0 = begin + t * BM;
    if (wave_key >= seq.s_len || row0 + BM <= wave_first) return;
    // every row of the tile sees every key of the wave: the first row's limit is the least
    const bool whole = row0 + BM <= rows && wave_key + 32 <= __builtin_amdgcn_readfirstlane(lds_limit[buf][0]);
    const U* summed = keys_role ? lds_q[buf] : lds_g[buf];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x16 s = zero16();
      kf.begin();
      if (keys_role) vf.begin();
      const int cols = again<kAgain>(lane) & 31;
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
        s = product<T>(read_cols<T, HDP, BM>(lds_q[buf], n * 32 + cols, st, half), kf.get(st), s);
      f32x16 p;
      if (keys_role) {
        f32x16 dp = zero16();
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
          dp = product<T>(read_cols<T, HDP, BM>(lds_g[buf], n * 32 + cols, st, half), vf.get(st), dp);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = n * 32 + acc_row(r, half);
          p[r] = exp2_fast(fmaf(s[r], c2, -lds_lse[buf][i]));
          s[r] = p[r] * (kFp16<T> ? (dp[r] - lds_delta[buf][i]) * range : dp[r] - lds_delta[buf][i]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = exp2_fast(fmaf(s[r], c2, -lds_lse[buf][n * 32 + acc_row(r, half)]));
      }
      if (!whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key >= lds_limit[buf][n * 32 + acc_row(r, half)]) s[r] = p[r] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = again<kAgain>(lane) & 63;
        if constexpr (!kRoles) {
          const Op<T> y = pack_rows<T>(p, u);
#pragma unroll
          for (int d = 0; d < DT; ++d)
            other[d] = product<T>(read_rows<T, HDP, BM>(lds_g[buf], n * 32, u, d * 32, at), y, other[d]);
        }
        const Op<T> x = pack_rows<T>(s, u);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          acc[d] = product<T>(read_rows<T, HDP, BM>(summed, n * 32, u, d * 32, at), x, acc[d]);
      }
    }
  };

  pass_tiles<BUFS>(max(0, (end - begin + BM - 1) / BM), fetch, place_tile, work);
  if (!live) return;
  const int64_t at = ((seq.s_off + key) * a.KV + kvh) * a.D;
  const float back = exp2_fast(-kLift<T>), f = keys_role ? a.scale * back / range : back;
  if (b.splits == 1)
    store_rows<T, DT>((keys_role ? dk : dv) + at, acc, f, a.D, half);
  else
    store_rows<float, DT>((keys_role ? pk : pv) + at, acc, f, a.D, half);
  if constexpr (!kRoles) {
    if (b.splits == 1)
      store_rows<T, DT>(dv + at, other, back, a.D, half);
    else
      store_rows<float, DT>(pv + at, other, back, a.D, half);
  }
}

// Adds the parts (planes `step` apart) in their order, four neighbouring elements a thread; blockIdx.y: which of two tensors, one
// plane behind the other.
template <typename T>
__global__ __launch_bounds__(256) void attn_backward_join_kernel(const float* part, int parts, int64_t step, int64_t plane,
                                                                 void* first, void* second) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= plane) return;
  const float* p = part + blockIdx.y * plane + i;
  T* out = static_cast<T*>(blockIdx.y == 0 ? first : second) + i;
  if (i + 4 <= plane) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) {
      float y[4];
      load_vec<float, 4>(p + s * step, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += y[j];
    }
    store_vec<T, 4>(out, x);
  } else {
    for (int j = 0; j < plane - i; ++j) {
      float x = 0.f;
      for (int s = 0; s < parts; ++s) x += p[s * step + j];
      out[j] = from_f32<T>(x);
    }
  }
}

// ---- launches ----------------------------------------------------------------------------------------------------------
// Parts of a key tile's rows: one workgroup fills a CU, so the parts are chosen that leave the fewest rows to walk in all rounds
// of the 256 CUs (777 keys on 3 key heads of 256, fp32, in 8 / 6 parts: 336 / 252 workgroups, 501 / 324 us), the
// more the better the balance: a causal tile at the start of a sequence has all the rows behind it (8192 tokens in 5 sequences,
// 16/4 heads of 128, bf16: 1 / 2 / 3 parts 468 / 269 / 263 us, and 13 / 18 us to join the parts; 8000 tokens, 4 heads of 64, fp32:
// 145 / 118 + 11 us).
int attn_backward_splits(int B, int64_t total_s, int KV, int D) {
  const int keys = attn_head_size(D) > 128 ? 64 : 128;
  const int64_t groups = std::max<int64_t>((ceil_div(total_s, keys) + B) * KV, 1);
  int best = 1;
  for (int parts = 2; parts <= 8 && groups * parts * keys <= 1024 * 128; ++parts)
    if (ceil_div(groups * parts, 256) * best <= ceil_div(groups * best, 256) * parts) best = parts;
  return best;
}

// Parts of a row tile's keys: where the row tiles leave compute units idle, into one workgroup a CU as far as every part of a
// sequence of the mean length keeps 128 keys (fp32) or 512 (16-bit types, whose tiles pass eight times as fast; the join is a
// launch).  Training, fp32, 11 sequences of 46 queries and 916 keys, one head of 192: 708 us whole, 436 / 365 / 335 us with 256 /
// 128 / 64 keys a part; one sequence of 761, one head of 256: 531 us, 395 / 313 / 291; bf16, 200 queries and 32768 keys, one head of
// 128: 1002 -> 168 us.
int attn_backward_q_splits(int dtype, int B, int64_t total_q, int64_t total_s, int KV, int G) {
  const int64_t groups = std::max<int64_t>((ceil_div(total_q * G, kAttnRows) + B) * KV, 1), mean = total_s / std::max(B, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({256 / groups, mean / (dtype == V3D_F32 ? 128 : 512), 16}));
}

inline size_t attn_backward_table(int64_t rows, int heads) { return align_up((size_t)rows * (size_t)heads * sizeof(float), 256); }

template <typename T, int HD>
int attn_backward_launch(AttnBwdArgs& b, hipStream_t stream, const char* what) {
  AttnArgs& a = b.f;
  const int64_t q_tiles = ceil_div(a.total_q * a.G, kAttnRows) + a.B;
  const int64_t s_tiles = ceil_div(a.total_s, 32 * kv_groups<T, HD>()) + a.B;
  int rc = attn_table_launch(a, const_cast<int64_t*>(a.table), kAttnRows, 32 * kv_groups<T, HD>(), stream, what);
  if (rc == 0 && kFp16<T> && a.total_s > 0) {
    const int64_t groups = std::min<int64_t>(ceil_div(a.total_s, 16), std::max(65536 / a.KV, 1));
    hipLaunchKernelGGL(attn_value_norm_kernel, dim3((unsigned)(groups * a.KV)), dim3(256), 0, stream, b);
    rc = launch_status(what);
  }
  if (rc == 0 && a.total_q > 0) {
    hipLaunchKernelGGL((attn_backward_q_kernel<T, HD>), dim3((unsigned)(q_tiles * a.KV * b.q_splits)), dim3(256), 0, stream, b);
    rc = launch_status(what);
    if (rc == 0 && b.q_splits > 1) {
      const int64_t plane = a.total_q * a.H * a.D;
      hipLaunchKernelGGL((attn_backward_join_kernel<T>), dim3((unsigned)ceil_div(plane, 1024)), dim3(256), 0, stream, b.part_q,
                         b.q_splits, plane, plane, b.dq, b.dq);
      rc = launch_status(what);
    }
  }
  if (rc == 0 && a.total_s > 0 && b.dk != nullptr) {
    hipLaunchKernelGGL((attn_backward_kv_kernel<T, HD>), dim3((unsigned)(s_tiles * a.KV * b.splits)),
                       dim3(kKvThreads), 0, stream, b);
    rc = launch_status(what);
    if (rc == 0 && b.splits > 1) {
      const int64_t plane = a.total_s * a.KV * a.D;
      hipLaunchKernelGGL((attn_backward_join_kernel<T>), dim3((unsigned)ceil_div(plane, 1024), 2), dim3(256), 0, stream, b.part,
                         b.splits, 2 * plane, plane, b.dk, b.dv);
      rc = launch_status(what);
    }
  }
  return rc;
}

template <typename T>
int attn_backward_type(AttnBwdArgs& b, hipStream_t stream, const char* what) {
  switch (attn_head_size(b.f.D)) {
    case 32: return attn_backward_launch<T, 32>(b, stream, what);
    case 64: return attn_backward_launch<T, 64>(b, stream, what);
    case 96: return attn_backward_launch<T, 96>(b, stream, what);
    case 128: return attn_backward_launch<T, 128>(b, stream, what);
    case 192: return attn_backward_launch<T, 192>(b, stream, what);
    default: return attn_backward_launch<T, 256>(b, stream, what);
  }
}

}  // namespace v3d

extern "C" {

size_t v3d_attention_pack_bwd_workspace_bytes(int B, int64_t total_q, int64_t total_s, int H, int KV, int D) {
  using namespace v3d;
  if (B < 0 || total_q < 0 || total_s < 0 || H <= 0 || KV <= 0 || H % KV != 0 || D <= 0) return 0;
  // delta and the rows' norms (of fp16 only, but the type is not asked for), the table, the parts
  const int splits = attn_backward_splits(B, total_s, KV, D), q_splits = attn_backward_q_splits(V3D_F32, B, total_q, total_s, KV, H / KV);
  return 2 * attn_backward_table(total_q, H) + attn_backward_table(total_s, KV) + attn_table_bytes(B, 4) +
         (q_splits > 1 ? align_up((size_t)q_splits * (size_t)total_q * (size_t)(H * D) * sizeof(float), 256) : 0) +
         (splits > 1 ? (size_t)splits * 2 * (size_t)total_s * (size_t)(KV * D) * sizeof(float) : 0);
}

int v3d_attention_pack_bwd(const void* grad, const void* q, const void* k, const void* v, const void* out,
                           const void* rest, const float* lse, const int64_t* q_lengths, const int64_t* s_lengths, void* grad_q,
                           void* grad_k, void* grad_v, int dtype, int B, int64_t total_q, int64_t total_s, int H, int KV,
                           int D, const int64_t* strides, float scale, int causal, void* workspace,
                           size_t workspace_bytes, int device, void* stream) {
  using namespace v3d;
  const char* what = "attention_pack_backward";
  int rc = attn_check(what, dtype, B, total_q, total_s, H, KV, D, scale);
  if (rc != 0) return rc;
  if (total_q == 0 && total_s == 0) return 0;
  V3D_REQUIRE(strides && (B == 0 || (q_lengths && s_lengths)), what, "null pointer");
  V3D_REQUIRE(total_q == 0 || (grad && q && out && lse), what, "null pointer");
  V3D_REQUIRE(total_s == 0 || (k && v), what, "null pointer");
  V3D_REQUIRE((grad_k == nullptr) == (grad_v == nullptr), what, "grad_k and grad_v come together");
  if (grad_q == nullptr && grad_k == nullptr) return 0;
  AttnBwdArgs b{};
  AttnArgs& a = b.f;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = const_cast<void*>(out);
  a.rest = dtype == V3D_F32 ? nullptr : const_cast<void*>(rest);
  a.lse = const_cast<float*>(lse);
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
  a.splits = 1;
  b.grad = grad;
  b.dq = grad_q;
  b.dk = grad_k;
  b.dv = grad_v;
  rc = attn_check_strides(what, a);
  if (rc != 0) return rc;
  const int keys = attn_head_size(D) > (dtype == V3D_F32 ? 96 : 128) ? 64 : 128;  // kv_groups
  if ((ceil_div(total_q * a.G, kAttnRows) + B) * KV > kAttnMaxGroups ||
      (ceil_div(total_s, keys) + B) * KV * attn_backward_splits(B, total_s, KV, D) > kAttnMaxGroups ||
      (attn_backward_splits(B, total_s, KV, D) > 1 && ceil_div(total_s * KV * D, 1024) > kAttnMaxGroups)) {
    set_last_error("%s: more than 2^24 row or key tiles (every sequence counts as one at least, once per key head)", what);
    return V3D_ERR_SIZE_LIMIT;
  }
  DeviceGuard guard(device);
  if (guard.rc != 0) return guard.rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Scratch ws;
  rc = ws.acquire(what, workspace, workspace_bytes,
                  v3d_attention_pack_bwd_workspace_bytes(B, total_q, total_s, H, KV, D), s);
  if (rc != 0) return rc;
  char* at = ws.base;
  auto take = [&](size_t bytes) {
    char* p = at;
    at += bytes;
    return reinterpret_cast<float*>(p);
  };
  b.delta = take(attn_backward_table(total_q, H));
  b.grad_norm = take(attn_backward_table(total_q, H));
  b.value_norm = take(attn_backward_table(total_s, KV));
  a.table = reinterpret_cast<int64_t*>(take(attn_table_bytes(B, 4)));
  const int q_splits = attn_backward_q_splits(V3D_F32, B, total_q, total_s, KV, a.G);  // the most of all types
  b.part_q = take(q_splits > 1 ? align_up((size_t)q_splits * (size_t)total_q * (size_t)(H * D) * sizeof(float), 256) : 0);
  b.part = reinterpret_cast<float*>(at);
  b.q_splits = grad_q == nullptr ? 1 : attn_backward_q_splits(dtype, B, total_q, total_s, KV, a.G);
  b.splits = attn_backward_splits(B, total_s, KV, D);
  rc = dtype == V3D_F32   ? attn_backward_type<float>(b, s, what)
       : dtype == V3D_F16 ? attn_backward_type<f16>(b, s, what)
                          : attn_backward_type<bf16>(b, s, what);
  return ws.release(what, rc);
}

}  // extern "C"
