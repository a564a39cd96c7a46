// attention_bwd.hip -- the gradients of attention_pack.
//
//   p_ij = exp(s_ij - lse_i),  dv_j = sum_i p_ij do_i,  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// Two kernels, each the owner of what it writes, so there are no atomics and the same input gives the same bits: one goes
// over the keys of a row tile (dq, and delta on the way), one over the rows of a key tile (dk, dv; the rows of all G query
// heads of a key head are folded, so the sum over a group needs nothing extra).  Both form s and dp again: 7 products
// instead of the 5 that the sums need, where a single kernel would add dq with atomics in fp32.
#include <algorithm>

#include "attn.h"

namespace v3d {

struct AttnBwdArgs {
  AttnArgs f;          // q, k, v, out, lse and the geometry of the forward (never a cache)
  const void* grad;    // (total_q, H, D) contiguous
  float* delta;        // (total_q, H): written by the dq kernel, read by the dk / dv kernel
  void* dq;            // (total_q, H, D), (total_s, KV, D) contiguous
  void* dk;
  void* dv;
};

template <typename T, int HD>
constexpr int bwd_keys() { return HD * (int)sizeof(T) > 256 ? 32 : 64; }

template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_backward_q_kernel(const AttnBwdArgs b) {
  constexpr int HDP = attn_pow2(HD);
  constexpr int BN = bwd_keys<T, HD>();
  constexpr int NT = BN / 32;
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int STEPS = HD / Mma<T>::kStep;
  constexpr int USTEPS = 32 / Mma<T>::kStep;
  constexpr int DT = HD / 32;
  typedef typename Mma<T>::Op Op;
  __shared__ T lds_k[BN * HDP];
  __shared__ T lds_v[BN * HDP];

  const AttnArgs& a = b.f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = lane >> 5;
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const AttnSeq seq = locate<kAttnRows, false>(a, id);
  T* dq = static_cast<T*>(b.dq);
  if (!seq.found) {  // rows behind the last sequence have no gradient
    const int64_t rows = (a.total_q - seq.q_end) * a.G;
    for (int i = threadIdx.x; i < kAttnRows; i += 256) {
      const int64_t r = seq.spare * kAttnRows + i;
      if (r >= rows) break;
      const int64_t at = (seq.q_end + r / a.G) * a.H + (int64_t)kvh * a.G + r % a.G;
      for (int d = 0; d < a.D; ++d) dq[at * a.D + d] = (T)0.f;
    }
    return;
  }
  const int rows = seq.q_len * a.G;
  if (seq.tile * kAttnRows >= rows) return;  // lengths that overrun the total were cut
  const int row = seq.tile * kAttnRows + wave * 32 + (lane & 31);
  const int token = min(row, rows - 1) / a.G;
  const int head = kvh * a.G + min(row, rows - 1) % a.G;
  auto limit_of = [&](int tok) {
    return a.causal ? max(0, min(seq.s_len, tok + seq.s_len - seq.q_len + 1)) : seq.s_len;
  };
  const int limit = limit_of(token);
  const bool wave_live = seq.tile * kAttnRows + wave * 32 < rows;
  const int wave_least = limit_of(min(seq.tile * kAttnRows + wave * 32, rows - 1) / a.G);
  const int wave_most = wave_live ? limit_of(min(seq.tile * kAttnRows + wave * 32 + 31, rows - 1) / a.G) : 0;
  const int most = limit_of(min(seq.tile * kAttnRows + kAttnRows - 1, rows - 1) / a.G);

  const T* q = static_cast<const T*>(a.q) + (seq.q_off + token) * a.q_row + (int64_t)head * a.q_head;
  const T* k = static_cast<const T*>(a.k) + seq.s_off * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + seq.s_off * a.v_row + (int64_t)kvh * a.v_head;
  const int64_t at = (seq.q_off + token) * a.H + head;
  const T* out = static_cast<const T*>(a.out) + at * a.D;
  const T* grad = static_cast<const T*>(b.grad) + at * a.D;

  Op qf[STEPS], gf[STEPS];
  float delta = 0.f;
#pragma unroll
  for (int st = 0; st < STEPS; ++st) {
    const int c0 = st * 2 * E + E * half;
    qf[st] = load_op<T>(q, c0, a.D, true);
    gf[st] = load_op<T>(grad, c0, a.D, true);
    const Op of = load_op<T>(out, c0, a.D, true);
#pragma unroll
    for (int j = 0; j < E; ++j) delta = fmaf((float)gf[st][j], (float)of[j], delta);
  }
  delta += __shfl_xor(delta, 32, 64);
  const float lse = a.lse[at];
  if (half == 0 && row < rows) b.delta[at] = delta;

  const float c2 = a.scale * kLog2e;
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = zero16();

  const int tiles = (most + BN - 1) / BN;
  for (int t = 0; t < tiles; ++t) {
    const int key0 = t * BN;
    __syncthreads();
    constexpr int CPR = HD / E;
    for (int i = threadIdx.x; i < BN * CPR; i += 256) {
      const int r = i / CPR, c = i % CPR;
      const bool live = key0 + r < seq.s_len;
      *reinterpret_cast<Chunk<T>*>(lds_k + tile_at<T, HDP>(r, c * E)) =
          load_chunk<T>(k + (int64_t)(key0 + r) * a.k_row, c * E, a.D, live);
      *reinterpret_cast<Chunk<T>*>(lds_v + tile_at<T, HDP>(r, c * E)) =
          load_chunk<T>(v + (int64_t)(key0 + r) * a.v_row, c * E, a.D, live);
    }
    __syncthreads();
    if (key0 >= wave_most) continue;
    const bool masked = key0 + BN > wave_least;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        s = Mma<T>::run(read_cols<T, HDP>(lds_k, n * 32 + (lane & 31), st, half), qf[st], s);
        dp = Mma<T>::run(read_cols<T, HDP>(lds_v, n * 32 + (lane & 31), st, half), gf[st], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_fast(fmaf(s[r], c2, -lse));
        const bool seen = !masked || key0 + n * 32 + acc_row(r, half) < limit;
        s[r] = seen ? p * (dp[r] - delta) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < USTEPS; ++u) {
        const Op ds = pack_rows<T>(s, u);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = Mma<T>::run(read_rows<T, HDP>(lds_k, n * 32, u, d * 32, lane), ds, acc[d]);
      }
    }
  }
  if (row >= rows) return;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = d * 32 + 8 * g + 4 * half + j;
        if (col < a.D) dq[at * a.D + col] = from_f32<T>(acc[d][g * 4 + j] * a.scale);
      }
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_backward_kv_kernel(const AttnBwdArgs b) {
  constexpr int HDP = attn_pow2(HD);
  constexpr int BM = bwd_keys<T, HD>();  // rows of a tile that passes by
  constexpr int NT = BM / 32;
  constexpr int E = 16 / (int)sizeof(T);
  constexpr int STEPS = HD / Mma<T>::kStep;
  constexpr int USTEPS = 32 / Mma<T>::kStep;
  constexpr int DT = HD / 32;
  typedef typename Mma<T>::Op Op;
  __shared__ T lds_q[BM * HDP];
  __shared__ T lds_g[BM * HDP];
  __shared__ float lds_lse[BM], lds_delta[BM];
  __shared__ int lds_limit[BM];

  const AttnArgs& a = b.f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = lane >> 5;
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const AttnSeq seq = locate<kAttnRows, true>(a, id);
  T* dk = static_cast<T*>(b.dk);
  T* dv = static_cast<T*>(b.dv);
  if (!seq.found) {
    for (int i = threadIdx.x; i < kAttnRows; i += 256) {
      const int64_t r = seq.s_end + seq.spare * kAttnRows + i;
      if (r >= a.total_s) break;
      for (int d = 0; d < a.D; ++d) dk[(r * a.KV + kvh) * a.D + d] = dv[(r * a.KV + kvh) * a.D + d] = (T)0.f;
    }
    return;
  }
  if (seq.tile * kAttnRows >= seq.s_len) return;  // cut
  const int key = seq.tile * kAttnRows + wave * 32 + (lane & 31);
  const bool live = key < seq.s_len;
  const int rows = seq.q_len * a.G;
  // rows that see the tile's first key: tokens from (first key) - (s_len - q_len) on
  const int key0 = seq.tile * kAttnRows;
  const int token0 = a.causal ? max(0, key0 - (seq.s_len - seq.q_len)) : 0;
  const int wave_key = key0 + wave * 32;
  const int wave_token0 = a.causal ? max(0, wave_key - (seq.s_len - seq.q_len)) : 0;

  const T* k = static_cast<const T*>(a.k) + (seq.s_off + min(key, seq.s_len - 1)) * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + (seq.s_off + min(key, seq.s_len - 1)) * a.v_row + (int64_t)kvh * a.v_head;
  Op kf[STEPS], vf[STEPS];
#pragma unroll
  for (int st = 0; st < STEPS; ++st) {
    kf[st] = load_op<T>(k, st * 2 * E + E * half, a.D, live);
    vf[st] = load_op<T>(v, st * 2 * E + E * half, a.D, live);
  }
  const float c2 = a.scale * kLog2e;
  f32x16 ak[DT], av[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) ak[d] = av[d] = zero16();

  const T* q = static_cast<const T*>(a.q) + seq.q_off * a.q_row + (int64_t)kvh * a.G * a.q_head;
  const T* grad = static_cast<const T*>(b.grad) + (seq.q_off * a.H + (int64_t)kvh * a.G) * a.D;
  const float* lse = a.lse + seq.q_off * a.H + kvh * a.G;
  const float* delta = b.delta + seq.q_off * a.H + kvh * a.G;

  for (int row0 = token0 * a.G / BM * BM; row0 < rows; row0 += BM) {
    __syncthreads();
    constexpr int CPR = HD / E;
    for (int i = threadIdx.x; i < BM * CPR; i += 256) {
      const int r = i / CPR, c = i % CPR;
      const bool in = row0 + r < rows;
      const int tok = min(row0 + r, rows - 1) / a.G, g = min(row0 + r, rows - 1) % a.G;
      *reinterpret_cast<Chunk<T>*>(lds_q + tile_at<T, HDP>(r, c * E)) =
          load_chunk<T>(q + tok * a.q_row + g * a.q_head, c * E, a.D, in);
      *reinterpret_cast<Chunk<T>*>(lds_g + tile_at<T, HDP>(r, c * E)) =
          load_chunk<T>(grad + ((int64_t)tok * a.H + g) * a.D, c * E, a.D, in);
    }
    if (threadIdx.x < BM) {
      const int r = row0 + threadIdx.x;
      const int tok = min(r, rows - 1) / a.G, g = min(r, rows - 1) % a.G;
      const int64_t i = (int64_t)tok * a.H + g;
      lds_lse[threadIdx.x] = lse[i];
      lds_delta[threadIdx.x] = delta[i];
      // keys that the row sees; a row past the last sees none
      lds_limit[threadIdx.x] = r >= rows ? 0 : a.causal ? max(0, min(seq.s_len, tok + seq.s_len - seq.q_len + 1)) : seq.s_len;
    }
    __syncthreads();
    if (wave_key >= seq.s_len || row0 + BM <= wave_token0 * a.G) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        s = Mma<T>::run(read_cols<T, HDP>(lds_q, n * 32 + (lane & 31), st, half), kf[st], s);
        dp = Mma<T>::run(read_cols<T, HDP>(lds_g, n * 32 + (lane & 31), st, half), vf[st], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = n * 32 + acc_row(r, half);
        const bool seen = key < lds_limit[i];
        const float p = exp2_fast(fmaf(s[r], c2, -lds_lse[i]));
        s[r] = seen ? p : 0.f;
        dp[r] = seen ? p * (dp[r] - lds_delta[i]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < USTEPS; ++u) {
        const Op p = pack_rows<T>(s, u), ds = pack_rows<T>(dp, u);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          av[d] = Mma<T>::run(read_rows<T, HDP>(lds_g, n * 32, u, d * 32, lane), p, av[d]);
          ak[d] = Mma<T>::run(read_rows<T, HDP>(lds_q, n * 32, u, d * 32, lane), ds, ak[d]);
        }
      }
    }
  }
  if (!live) return;
  const int64_t at = ((seq.s_off + key) * a.KV + kvh) * a.D;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = d * 32 + 8 * g + 4 * half + j;
        if (col < a.D) {
          dk[at + col] = from_f32<T>(ak[d][g * 4 + j] * a.scale);
          dv[at + col] = from_f32<T>(av[d][g * 4 + j]);
        }
      }
}

// ---- launches ----------------------------------------------------------------------------------------------------------
template <typename T, int HD>
int attn_backward_launch(const AttnBwdArgs& b, hipStream_t stream, const char* what) {
  const AttnArgs& a = b.f;
  const int64_t q_tiles = ceil_div(a.total_q * a.G, kAttnRows) + a.B, s_tiles = ceil_div(a.total_s, kAttnRows) + a.B;
  int rc = 0;
  if (a.total_q > 0) {
    hipLaunchKernelGGL((attn_backward_q_kernel<T, HD>), dim3((unsigned)(q_tiles * a.KV)), dim3(256), 0, stream, b);
    rc = launch_status(what);
  }
  if (rc == 0 && a.total_s > 0) {
    hipLaunchKernelGGL((attn_backward_kv_kernel<T, HD>), dim3((unsigned)(s_tiles * a.KV)), dim3(256), 0, stream, b);
    rc = launch_status(what);
  }
  return rc;
}

template <typename T>
int attn_backward_type(const AttnBwdArgs& b, hipStream_t stream, const char* what) {
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
  (void)B;
  (void)total_s;
  (void)KV;
  (void)D;
  return total_q > 0 && H > 0 ? (size_t)total_q * (size_t)H * sizeof(float) : 0;
}

int v3d_attention_pack_bwd(const void* grad, const void* q, const void* k, const void* v, const void* out,
                           const float* lse, const int64_t* q_lengths, const int64_t* s_lengths, void* grad_q,
                           void* grad_k, void* grad_v, int dtype, int B, int64_t total_q, int64_t total_s, int H, int KV,
                           int D, const int64_t* strides, float scale, int causal, void* workspace,
                           size_t workspace_bytes, int device, void* stream) {
  using namespace v3d;
  const char* what = "attention_pack_backward";
  int rc = attn_check(what, dtype, B, total_q, total_s, H, KV, D, scale);
  if (rc != 0) return rc;
  if (total_q == 0 && total_s == 0) return 0;
  V3D_REQUIRE(strides && (B == 0 || (q_lengths && s_lengths)), what, "null pointer");
  V3D_REQUIRE(total_q == 0 || (grad && q && out && lse && grad_q), what, "null pointer");
  V3D_REQUIRE(total_s == 0 || (k && v && grad_k && grad_v), what, "null pointer");
  DeviceGuard guard(device);
  if (guard.rc != 0) return guard.rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  AttnBwdArgs b{};
  AttnArgs& a = b.f;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = const_cast<void*>(out);
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
  a.H = H;
  a.KV = KV;
  a.G = H / KV;
  a.D = D;
  a.scale = scale;
  a.causal = causal;
  a.splits = 1;
  b.grad = grad;
  b.dq = grad_q;
  b.dk = grad_k;
  b.dv = grad_v;
  Scratch ws;
  rc = ws.acquire(what, workspace, workspace_bytes,
                  v3d_attention_pack_bwd_workspace_bytes(B, total_q, total_s, H, KV, D), s);
  if (rc != 0) return rc;
  b.delta = reinterpret_cast<float*>(ws.base);
  rc = dtype == V3D_F32   ? attn_backward_type<float>(b, s, what)
       : dtype == V3D_F16 ? attn_backward_type<f16>(b, s, what)
                          : attn_backward_type<bf16>(b, s, what);
  return ws.release(what, rc);
}

}  // extern "C"
