// attention.hip -- softmax attention inside the sequences of a pack, and of new tokens against cached keys and values.
//
//   s_ij = scale * q_i . k_j over the keys that query i sees,  o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// Rows: the G = H / KV query heads of a key head are folded into the rows of that head's products (row = token * G + head),
// so grouped heads read every key once per tile whatever G is, and a single token of 8 heads fills 8 columns of a product
// instead of one.
#include <algorithm>

#include "attn.h"

namespace v3d {

// Keys of a tile: two tiles of keys and values (one worked on, one arriving) stay within 64 KiB up to 512-byte rows, so that
// two workgroups share a CU.
template <typename T, int HD>
constexpr int attn_keys() { return HD * (int)sizeof(T) > 256 ? 32 : 64; }

template <typename T, int HD>
__global__ __launch_bounds__(256, HD * sizeof(T) <= 256 ? 2 : 1) void attn_forward_kernel(const AttnArgs a) {
  constexpr int HDP = attn_pow2(HD);
  constexpr int BN = attn_keys<T, HD>();
  constexpr int NT = BN / 32;                       // 32-key blocks of a tile
  constexpr int STEPS = HD / Mma<T>::kStep;         // product steps over the head size
  constexpr int USTEPS = 32 / Mma<T>::kStep;        // product steps over a 32-key block
  constexpr int DT = HD / 32;
  typedef typename Mma<T>::Op Op;
  __shared__ T lds_k[2][BN * HDP];
  __shared__ T lds_v[2][BN * HDP];
  __shared__ int lds_bad[2];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = lane >> 5;
  int64_t id = blockIdx.x;
  const int kvh = (int)(id % a.KV);
  id /= a.KV;
  const int split = (int)(id % a.splits);
  id = (int64_t)(gridDim.x / (a.KV * a.splits)) - 1 - id / a.splits;  // causal: the longest tiles of a sequence start first
  const AttnSeq seq = locate_rows<kAttnRows>(a, id);
  if (!seq.found) {  // the launch covers a bound: the rest of it clears the rows behind the last sequence
    if (a.capacity == 0 && split == 0) {
      const int64_t rows = (a.total_q - seq.q_end) * a.G;
      for (int i = threadIdx.x; i < kAttnRows; i += 256) {
        const int64_t r = seq.spare * kAttnRows + i;
        if (r >= rows) break;
        const int64_t at = (seq.q_end + r / a.G) * a.H + (int64_t)kvh * a.G + r % a.G;
        for (int d = 0; d < a.D; ++d) static_cast<T*>(a.out)[at * a.D + d] = (T)0.f;
        if (a.lse) a.lse[at] = -__builtin_inff();
      }
    }
    return;
  }
  const int rows = seq.q_len * a.G;
  if (seq.tile * kAttnRows >= rows) return;  // lengths that overrun the total were cut
  const int row = seq.tile * kAttnRows + wave * 32 + (lane & 31);
  const int token = div_g(a, min(row, rows - 1));
  const int head = kvh * a.G + min(row, rows - 1) - token * a.G;
  const int limit = attn_limit(a, seq, token);  // this lane's query sees keys [0, limit)
  // the wave's and the workgroup's first and last rows bound what they have to look at
  const bool wave_live = seq.tile * kAttnRows + wave * 32 < rows;
  const int wave_least = __builtin_amdgcn_readfirstlane(limit);
  const int wave_most = wave_live ? attn_limit(a, seq, div_g(a, min(seq.tile * kAttnRows + wave * 32 + 31, rows - 1))) : 0;
  const int most = attn_limit(a, seq, div_g(a, min(seq.tile * kAttnRows + kAttnRows - 1, rows - 1)));
  const int least = attn_limit(a, seq, div_g(a, min(seq.tile * kAttnRows, rows - 1)));

  const int tiles = (most + BN - 1) / BN;
  const int per_split = (tiles + a.splits - 1) / a.splits;
  const int t_begin = split * per_split, t_end = min(tiles, t_begin + per_split);

  const int token0 = div_g(a, seq.tile * kAttnRows);
  const T* q = static_cast<const T*>(a.q) + (seq.q_off + token0) * a.q_row + (int64_t)kvh * a.G * a.q_head;
  const T* k = static_cast<const T*>(a.k) + seq.b * a.k_batch + seq.s_off * a.k_row + (int64_t)kvh * a.k_head;
  const T* v = static_cast<const T*>(a.v) + seq.b * a.v_batch + seq.s_off * a.v_row + (int64_t)kvh * a.v_head;

  Op qf[STEPS];
  load_ops<T>(qf, q, (token - token0) * (int)a.q_row + (head - kvh * a.G) * (int)a.q_head, half, a.D);

  // The tile after the one that is worked on is on its way in registers meanwhile.
  TileStage<T, HD, BN> stage_k, stage_v;
  if (threadIdx.x < 2) lds_bad[threadIdx.x] = 0;
  auto fetch = [&](int t) {
    stage_k.fetch(k + (int64_t)t * BN * a.k_row, a.k_row, a.D, seq.s_len - t * BN);
    stage_v.fetch(v + (int64_t)t * BN * a.v_row, a.v_row, a.D, seq.s_len - t * BN);
  };
  auto place_tile = [&](int t, int buf) {
    stage_k.store(lds_k[buf], a.D);
    stage_v.store(lds_v[buf], a.D);
    // values of a tile that some query sees in part: see below
    if (t * BN + BN > least && stage_v.nonfinite()) lds_bad[buf] = t + 1;
  };

  const float c2 = a.scale * kLog2e;
  float m = -__builtin_inff(), l = 0.f;  // running maximum of scale * log2(e) * score, and the sum of 2^(that - m)
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = zero16();

  auto work = [&](int t, auto buffer) {
    constexpr int buf = decltype(buffer)::value;
    const int key0 = t * BN;
    const bool active = key0 < wave_most;
    f32x16 s[NT];
    if (active) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n] = zero16();
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          s[n] = Mma<T>::run(read_cols<T, HDP>(lds_k[buf], n * 32 + (lane & 31), st, half), qf[st], s[n]);
      if (key0 + BN > wave_least) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (key0 + n * 32 + acc_row(r, half) >= limit) s[n][r] = -__builtin_inff();
      }
      // maximum of the lane, then with the lane that holds the other keys of this query
      float top = -__builtin_inff();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
      top = halves_max(top) * c2;
      // The maximum moves only when a probability would exceed 2^8: what was summed is rescaled rarely, and a stale
      // maximum costs no accuracy (16-bit probabilities keep their relative precision up to 2^8, the sums are fp32).
      if (__any(top > m + 8.f)) {
        const float m_new = fmaxf(m, top);
        const float alpha = m_new == -__builtin_inff() ? 1.f : exp2_fast(m - m_new);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      const float base = m == -__builtin_inff() ? 0.f : m;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[n][r] = exp2_fast(fmaf(s[n][r], c2, -base));
          sum += s[n][r];
        }
      l += sum;
    }
    if (lds_bad[buf] == t + 1) {
      // An infinity or NaN among the values of a tile that some query sees in part must not reach the queries that do not
      // see it (0 * inf).  It is added key by key to the queries that do, then cleared for the product.  The probabilities
      // wait in the keys' place, which nobody reads any more.
      __syncthreads();
      T* lds_p = lds_k[buf] + wave * (BN * 32);
      if (active) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) lds_p[(n * 32 + acc_row(r, half)) * 32 + (lane & 31)] = from_f32<T>(s[n][r]);
      }
      __syncthreads();
      if (active) {
#pragma unroll 1
        for (int key = 0; key < BN && key0 + key < wave_most; ++key) {
          const float p = to_f32(lds_p[key * 32 + (lane & 31)]);
          const bool seen = key0 + key < limit;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float w = to_f32(lds_v[buf][tile_at<T, HDP>(key, d * 32 + acc_row(r, half))]);
              if (seen && !(__builtin_fabsf(w) < __builtin_inff())) o[d][r] += p * w;
            }
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < BN * HDP; i += 256)
        if (!(__builtin_fabsf(to_f32(lds_v[buf][i])) < __builtin_inff())) lds_v[buf][i] = (T)0.f;
      __syncthreads();
    }
    if (active) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int u = 0; u < USTEPS; ++u) {
          const Op p = pack_rows<T>(s[n], u);
#pragma unroll
          for (int d = 0; d < DT; ++d)
            o[d] = Mma<T>::run(read_rows<T, HDP>(lds_v[buf], n * 32, u, d * 32, lane), p, o[d]);
        }
    }
  };

  if (t_begin < t_end) {
    __syncthreads();  // lds_bad
    fetch(t_begin);
    place_tile(t_begin, 0);
    __syncthreads();
    for (int t = t_begin; t < t_end; t += 2) {
      if (t + 1 < t_end) fetch(t + 1);
      work(t, Const<0>{});
      if (t + 1 < t_end) place_tile(t + 1, 1);
      __syncthreads();
      if (t + 1 >= t_end) break;
      if (t + 2 < t_end) fetch(t + 2);
      work(t + 1, Const<1>{});
      if (t + 2 < t_end) place_tile(t + 2, 0);
      __syncthreads();
    }
  }

  l = halves_sum(l);
  if (row >= rows) return;
  if (a.splits == 1) {
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN sum stays a NaN
    const int64_t at = (seq.q_off + token) * a.H + head;
    store_rows<T, DT>(static_cast<T*>(a.out) + at * a.D, o, inv, a.D, half);
    if (a.lse && half == 0) a.lse[at] = l == 0.f ? -__builtin_inff() : m + log2f(l);
    return;
  }
  const int64_t part = (((int64_t)id * a.KV + kvh) * a.splits + split) * kAttnRows + wave * 32 + (lane & 31);
  store_rows<float, DT>(a.part_o + part * a.D, o, 1.f, a.D, half);
  if (half == 0) {
    a.part_ml[part * 2] = m;
    a.part_ml[part * 2 + 1] = l;
  }
}

// Joins the parts of a row tile's keys: one wave per row, lanes over the columns.
template <typename T, int TILE>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
  float m = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[(part + (int64_t)s * TILE) * 2]);
  const float base = m == -__builtin_inff() ? 0.f : m;
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const int64_t p = part + (int64_t)s * TILE;
    const float f = exp2_fast(a.part_ml[p * 2] - base);
    l = fmaf(a.part_ml[p * 2 + 1], f, l);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 64 * j < a.D) o[j] = fmaf(a.part_o[p * a.D + lane + 64 * j], f, o[j]);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int token = div_g(a, row);
  const int64_t out = (seq.q_off + token) * a.H + (int64_t)kvh * a.G + row - token * a.G;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < a.D) static_cast<T*>(a.out)[out * a.D + lane + 64 * j] = from_f32<T>(o[j] * inv);
  if (a.lse && lane == 0) a.lse[out] = l == 0.f ? -__builtin_inff() : m + log2f(l);
}

// ---- launches ----------------------------------------------------------------------------------------------------------
struct AttnPlan {
  int64_t tiles;    // row tiles (a bound in a pack)
  int splits;
  size_t bytes;     // workspace
};

inline AttnPlan attn_plan(int B, int64_t total_q, int64_t longest, int tokens, int KV, int G, int D) {
  AttnPlan p;
  p.tiles = tokens > 0 ? B * ceil_div((int64_t)tokens * G, kAttnRows) : ceil_div(total_q * G, kAttnRows) + B;
  const int64_t groups = p.tiles * KV;
  // keys are divided only where the row tiles leave compute units idle; a part has at least 4 key tiles of the bound
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(groups, 1), longest / 256));
  p.splits = std::min(p.splits, 64);
  p.bytes = p.splits > 1 ? (size_t)(groups * p.splits * kAttnRows) * (size_t)(D + 2) * sizeof(float) : 0;
  return p;
}

template <typename T, int HD>
int attn_forward_launch(const AttnArgs& a, int64_t tiles, hipStream_t stream, const char* what) {
  hipLaunchKernelGGL((attn_forward_kernel<T, HD>), dim3((unsigned)(tiles * a.KV * a.splits)), dim3(256), 0, stream, a);
  int rc = launch_status(what);
  if (rc == 0 && a.splits > 1) {
    hipLaunchKernelGGL((attn_join_kernel<T, kAttnRows>), dim3((unsigned)(tiles * a.KV * (kAttnRows / 4))), dim3(256), 0,
                       stream, a);
    rc = launch_status(what);
  }
  return rc;
}

template <typename T>
int attn_forward_type(const AttnArgs& a, int64_t tiles, hipStream_t stream, const char* what) {
  switch (attn_head_size(a.D)) {
    case 32: return attn_forward_launch<T, 32>(a, tiles, stream, what);
    case 64: return attn_forward_launch<T, 64>(a, tiles, stream, what);
    case 96: return attn_forward_launch<T, 96>(a, tiles, stream, what);
    case 128: return attn_forward_launch<T, 128>(a, tiles, stream, what);
    case 192: return attn_forward_launch<T, 192>(a, tiles, stream, what);
    default: return attn_forward_launch<T, 256>(a, tiles, stream, what);
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
// 129 tokens and the heads of a group of a query tensor.
int attn_check_strides(const char* what, const AttnArgs& a) {
  const int64_t reach = (int64_t)1 << 29;  // elements of 4 bytes
  auto fits = [&](int64_t row, int64_t head) {
    return row >= 0 && head >= 0 && row < reach / 130 && head < reach / (2 * a.G) && 129 * row + a.G * head + a.D < reach;
  };
  if (!fits(a.q_row, a.q_head) || !fits(a.k_row, 0) || !fits(a.v_row, 0) || !fits((int64_t)a.H * a.D, a.D)) {
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
  if (plan.tiles * a.KV * plan.splits > ((int64_t)1 << 31) / 64) {
    set_last_error("%s: too many tiles", what);
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
    a.part_o = reinterpret_cast<float*>(ws.base);
    a.part_ml = a.part_o + plan.tiles * a.KV * a.splits * kAttnRows * a.D;
  }
  int rc = dtype == V3D_F32   ? attn_forward_type<float>(a, plan.tiles, s, what)
           : dtype == V3D_F16 ? attn_forward_type<f16>(a, plan.tiles, s, what)
                              : attn_forward_type<bf16>(a, plan.tiles, s, what);
  return ws.release(what, rc);
}

}  // namespace v3d

extern "C" {

size_t v3d_attention_pack_workspace_bytes(int B, int64_t total_q, int64_t total_s, int H, int KV, int D) {
  if (B <= 0 || total_q <= 0 || H <= 0 || KV <= 0 || H % KV != 0 || D <= 0) return 0;
  return v3d::attn_plan(B, total_q, total_s, 0, KV, H / KV, D).bytes;
}

int v3d_attention_pack_fwd(const void* q, const void* k, const void* v, const int64_t* q_lengths,
                           const int64_t* s_lengths, void* out, float* lse, int dtype, int B, int64_t total_q,
                           int64_t total_s, int H, int KV, int D, const int64_t* strides, float scale, int causal,
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
