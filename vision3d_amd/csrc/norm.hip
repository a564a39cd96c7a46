// norm.hip -- layer normalisation of rows, optionally of the sum of two inputs (post-norm layer), and its backward.
//
//   t = x + r,  mean = sum(t) / C,  var = sum((t - mean)^2) / C,  rstd = 1 / sqrt(var + eps),  u = (t - mean) * rstd
//   y = u * w + b
//   dt = rstd * (gw - sum(gw) / C - u * sum(gw * u) / C)  with gw = g * w;  dx = dr = dt
//   dw = sum over rows of g * u,  db = sum over rows of g
//
// Bound: HBM.  Forward reads x (and r) and writes y once; backward reads x (and r) and g and writes dt once: the sum t is
// formed again instead of being kept, which costs a second read of r where keeping it would cost a write and a read.
// TPR threads hold a whole row in registers (NIT vectors of 16 bytes each), so the variance is the centred one from a
// single read.  The column sums of the backward stay in registers over all the rows that a thread visits, are joined per
// workgroup in LDS and leave as one partial row per workgroup; a second small kernel adds the partial rows in a fixed
// order.  No atomics: the same input gives the same bits.  Rows start at any element: 16-byte accesses need no alignment.
//
// Measured (a large copy moves 4.9 TB/s): 120000 x 256 fp32 with residual 67 us = 5.5 TB/s; 65536 x 1024 bf16 with residual,
// forward 78 us = 5.2 TB/s, backward 101 + 7 us = 5.3 TB/s; 20011 x 771 fp16, forward 24, backward 30 + 7 us.
#include <algorithm>

#include "common.h"
#include "numeric.h"

namespace v3d {

constexpr int kNormThreads = 256;

struct NormArgs {
  const void* x;
  const void* r;       // or NULL
  const void* w;       // or NULL = 1
  const void* b;       // or NULL = 0
  const void* g;       // backward: gradient of y
  void* y;             // forward: y; backward: dt
  float* mean;
  float* rstd;
  float* partial;      // backward: (2, gridDim.x, C) partial column sums, or NULL
  int64_t rows;
  int C;
  float eps;
};

// Sum over the TPR threads of a row, handed to all of them.  Rows of more than a wave meet in LDS; `slot` alternates so
// that one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds, int& slot) {
  if constexpr (TPR <= 64) {
    return lanes_sum<TPR>(v);
  } else {
    constexpr int W = TPR / 64;
    v = lanes_sum<64>(v);
    float* at = lds + slot * 16;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) s += at[k];
    return s;
  }
}

// The vector of columns [c0, c0 + VEC) of a row; columns from C on read as zeros.
template <typename T, int VEC>
__device__ __forceinline__ void load_cols(const T* row, int c0, int C, float (&out)[VEC]) {
  if (c0 + VEC <= C) {
    load_vec<T, VEC>(row + c0, out);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = c0 + j < C ? to_f32(row[c0 + j]) : 0.f;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_cols(T* row, int c0, int C, const float (&in)[VEC]) {
  if (c0 + VEC <= C) {
    store_vec<T, VEC>(row + c0, in);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c0 + j < C) row[c0 + j] = from_f32<T>(in[j]);
  }
}

template <typename T, typename TW, int TPR, int NIT>
__global__ __launch_bounds__(TPR > 256 ? TPR : kNormThreads) void norm_forward_kernel(const NormArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kBlock = TPR > 256 ? TPR : kNormThreads;
  constexpr int RPB = kBlock / TPR;  // rows per workgroup at a time
  __shared__ float lds[32];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int C = a.C;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  float w[NIT][VEC], b[NIT][VEC];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int c0 = (i * TPR + t) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = a.w == nullptr ? 1.f : 0.f;
      b[i][j] = 0.f;
    }
    if (a.w != nullptr) load_cols<TW, VEC>(static_cast<const TW*>(a.w), c0, C, w[i]);
    if (a.b != nullptr) load_cols<TW, VEC>(static_cast<const TW*>(a.b), c0, C, b[i]);
  }
  const float inv = 1.f / (float)C;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row - threadIdx.x / TPR < a.rows;
       row += (int64_t)gridDim.x * RPB) {
    const bool live = row < a.rows;  // idle rows of the last round still take part in the sums' barriers
    const int64_t at = (live ? row : 0) * C;
    float v[NIT][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      load_cols<T, VEC>(x + at, (i * TPR + t) * VEC, C, v[i]);
      if (r != nullptr) {
        float e[VEC];
        load_cols<T, VEC>(r + at, (i * TPR + t) * VEC, C, e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += e[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[i][j];
    }
    const float mean = row_sum<TPR>(s, lds, slot) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = v[i][j] - mean;
        if ((i * TPR + t) * VEC + j < C) s = fmaf(d, d, s);
        v[i][j] = d;
      }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(s, lds, slot) * inv + a.eps);
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[i][j], b[i][j]);
      store_cols<T, VEC>(static_cast<T*>(a.y) + at, (i * TPR + t) * VEC, C, v[i]);
    }
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename TW, int TPR, int NIT>
__global__ __launch_bounds__(TPR > 256 ? TPR : kNormThreads) void norm_backward_kernel(const NormArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kBlock = TPR > 256 ? TPR : kNormThreads;
  constexpr int RPB = kBlock / TPR;
  constexpr int kCols = TPR * NIT * VEC;
  __shared__ float lds[32];
  __shared__ float join[RPB > 1 ? 2 * kCols : 1];
  int slot = 0;
  const int t = threadIdx.x % TPR;
  const int C = a.C;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  const T* g = static_cast<const T*>(a.g);
  float w[NIT][VEC], dw[NIT][VEC], db[NIT][VEC];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[i][j] = 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
    if (a.w != nullptr) load_cols<TW, VEC>(static_cast<const TW*>(a.w), (i * TPR + t) * VEC, C, w[i]);
  }
  const float inv = 1.f / (float)C;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row - threadIdx.x / TPR < a.rows;
       row += (int64_t)gridDim.x * RPB) {
    const bool live = row < a.rows;
    const int64_t at = (live ? row : 0) * C;
    const float mean = a.mean[live ? row : 0], rstd = a.rstd[live ? row : 0];
    float u[NIT][VEC], gw[NIT][VEC];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int c0 = (i * TPR + t) * VEC;
      load_cols<T, VEC>(x + at, c0, C, u[i]);
      load_cols<T, VEC>(g + at, c0, C, gw[i]);
      if (r != nullptr) {
        float e[VEC];
        load_cols<T, VEC>(r + at, c0, C, e);
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[i][j] += e[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {  // columns from C on: gw = 0, so u there adds nothing
        u[i][j] = (u[i][j] - mean) * rstd;
        if (live && c0 + j < C) {
          dw[i][j] = fmaf(gw[i][j], u[i][j], dw[i][j]);
          db[i][j] += gw[i][j];
        }
        gw[i][j] *= w[i][j];
        s1 += gw[i][j];
        s2 = fmaf(gw[i][j], u[i][j], s2);
      }
    }
    s1 = row_sum<TPR>(s1, lds, slot) * inv;
    s2 = row_sum<TPR>(s2, lds, slot) * inv;
    if (!live || a.y == nullptr) continue;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) gw[i][j] = (gw[i][j] - s1 - u[i][j] * s2) * rstd;
      store_cols<T, VEC>(static_cast<T*>(a.y) + at, (i * TPR + t) * VEC, C, gw[i]);
    }
  }
  if (a.partial == nullptr) return;
  float* pw = a.partial + (int64_t)blockIdx.x * C;
  float* pb = pw + (int64_t)gridDim.x * C;
  if constexpr (RPB > 1) {  // the workgroup's row slots, one after another (a fixed order)
    for (int k = 0; k < RPB; ++k) {
      if ((int)threadIdx.x / TPR == k) {
#pragma unroll
        for (int i = 0; i < NIT; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = (i * VEC + j) * TPR + t;  // any one-to-one place
            join[c] = k == 0 ? dw[i][j] : join[c] + dw[i][j];
            join[kCols + c] = k == 0 ? db[i][j] : join[kCols + c] + db[i][j];
          }
      }
      __syncthreads();
    }
    if ((int)threadIdx.x / TPR != 0) return;
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        dw[i][j] = join[(i * VEC + j) * TPR + t];
        db[i][j] = join[kCols + (i * VEC + j) * TPR + t];
      }
  }
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    store_cols<float, VEC>(pw, (i * TPR + t) * VEC, C, dw[i]);
    store_cols<float, VEC>(pb, (i * TPR + t) * VEC, C, db[i]);
  }
}

// dw[c] / db[c] = the sum of the partial rows: 16 columns x 64 row groups per workgroup, joined by a tree in LDS.
template <typename TW>
__global__ __launch_bounds__(1024) void norm_columns_kernel(const float* __restrict__ partial, int parts, int C, TW* dw,
                                                            TW* db) {
  __shared__ float lds[64][17];
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + col;
  const float* p = partial + (int64_t)blockIdx.y * parts * C;
  float s = 0.f;
  if (c < C)
    for (int k = grp; k < parts; k += 64) s += p[(int64_t)k * C + c];
  lds[grp][col] = s;
  __syncthreads();
  for (int half = 32; half >= 1; half >>= 1) {
    if (grp < half) lds[grp][col] += lds[grp + half][col];
    __syncthreads();
  }
  TW* out = blockIdx.y == 0 ? dw : db;
  if (grp == 0 && c < C && out != nullptr) out[c] = from_f32<TW>(lds[0][col]);
}

// ---- launches ----------------------------------------------------------------------------------------------------------
// The geometry goes by the row's length alone: the fewest threads that hold it in at most 2 vectors each (the backward
// carries five values per column: 80 registers with 2 vectors of 8).
constexpr int kNormMaxParts = 1024;

inline int norm_max_channels(int dtype) { return dtype == V3D_F32 ? V3D_NORM_MAX_CHANNELS / 2 : V3D_NORM_MAX_CHANNELS; }

// Workgroups of the backward: enough to fill 256 CUs, few enough that the partial rows stay small beside the input.
inline int norm_parts(int64_t rows, int rows_per_block) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(kNormMaxParts, ceil_div(rows, (int64_t)rows_per_block)));
}

template <typename T, typename TW, int TPR, int NIT>
int norm_launch(const NormArgs& a, bool backward, void* dw, void* db, hipStream_t stream, const char* what) {
  constexpr int block = TPR > 256 ? TPR : kNormThreads;
  constexpr int rpb = block / TPR;
  if (!backward) {
    const int64_t groups = std::min<int64_t>(ceil_div(a.rows, (int64_t)rpb), 8192);
    hipLaunchKernelGGL((norm_forward_kernel<T, TW, TPR, NIT>), dim3((unsigned)groups), dim3(block), 0, stream, a);
    return launch_status(what);
  }
  const int parts = norm_parts(a.rows, rpb);
  hipLaunchKernelGGL((norm_backward_kernel<T, TW, TPR, NIT>), dim3(parts), dim3(block), 0, stream, a);
  int rc = launch_status(what);
  if (rc == 0 && a.partial != nullptr) {
    hipLaunchKernelGGL((norm_columns_kernel<TW>), dim3((unsigned)ceil_div(a.C, 16), 2), dim3(1024), 0, stream, a.partial,
                       parts, a.C, static_cast<TW*>(dw), static_cast<TW*>(db));
    rc = launch_status(what);
  }
  return rc;
}

template <typename T, typename TW>
int norm_dispatch(const NormArgs& a, bool backward, void* dw, void* db, hipStream_t stream, const char* what) {
  constexpr int VEC = 16 / sizeof(T);
  const int vecs = (int)ceil_div(a.C, VEC);
  if (vecs <= 16) return norm_launch<T, TW, 16, 1>(a, backward, dw, db, stream, what);
  if (vecs <= 32) return norm_launch<T, TW, 32, 1>(a, backward, dw, db, stream, what);
  if (vecs <= 64) return norm_launch<T, TW, 64, 1>(a, backward, dw, db, stream, what);
  if (vecs <= 128) return norm_launch<T, TW, 64, 2>(a, backward, dw, db, stream, what);
  if (vecs <= 256) return norm_launch<T, TW, 256, 1>(a, backward, dw, db, stream, what);
  if (vecs <= 512) return norm_launch<T, TW, 256, 2>(a, backward, dw, db, stream, what);
  if (vecs <= 1024) return norm_launch<T, TW, 1024, 1>(a, backward, dw, db, stream, what);
  return norm_launch<T, TW, 1024, 2>(a, backward, dw, db, stream, what);
}

int norm_run(const NormArgs& a, int dtype, int wdtype, bool backward, void* dw, void* db, hipStream_t stream,
             const char* what) {
  if (dtype == V3D_F32) return norm_dispatch<float, float>(a, backward, dw, db, stream, what);
  if (dtype == V3D_F16)
    return wdtype == V3D_F32 ? norm_dispatch<f16, float>(a, backward, dw, db, stream, what)
                             : norm_dispatch<f16, f16>(a, backward, dw, db, stream, what);
  return wdtype == V3D_F32 ? norm_dispatch<bf16, float>(a, backward, dw, db, stream, what)
                           : norm_dispatch<bf16, bf16>(a, backward, dw, db, stream, what);
}

int norm_check(const char* what, int dtype, int wdtype, int64_t rows, int64_t C, float eps) {
  V3D_REQUIRE(dtype == V3D_F32 || dtype == V3D_F16 || dtype == V3D_BF16, what, "unknown element type");
  V3D_REQUIRE(wdtype == dtype || wdtype == V3D_F32, what, "weights are of the features' type or fp32");
  V3D_REQUIRE(rows >= 0 && C >= 1, what, "bad shape");
  V3D_REQUIRE(eps >= 0.f, what, "eps must not be negative");
  if (C > norm_max_channels(dtype)) {
    set_last_error("%s: %lld channels, at most %d of this type", what, (long long)C, norm_max_channels(dtype));
    return V3D_ERR_SIZE_LIMIT;
  }
  return 0;
}

}  // namespace v3d

extern "C" {

int v3d_layer_norm_fwd(const void* feats, const void* residual, const void* weight, const void* bias, void* out,
                       float* mean, float* rstd, int dtype, int weight_dtype, int64_t rows, int64_t C, float eps,
                       int device, void* stream) {
  using namespace v3d;
  const char* what = "layer_norm";
  int rc = norm_check(what, dtype, weight_dtype, rows, C, eps);
  if (rc != 0) return rc;
  V3D_REQUIRE((mean == nullptr) == (rstd == nullptr), what, "mean and rstd come together");
  if (rows == 0) return 0;
  V3D_REQUIRE(feats && out, what, "null pointer");
  DeviceGuard guard(device);
  if (guard.rc != 0) return guard.rc;
  NormArgs a{feats, residual, weight, bias, nullptr, out, mean, rstd, nullptr, rows, (int)C, eps};
  return norm_run(a, dtype, weight_dtype, false, nullptr, nullptr, static_cast<hipStream_t>(stream), what);
}

size_t v3d_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0) return 0;
  // at most kNormMaxParts partial rows of two sums, and no more than there are rows
  return (size_t)std::min<int64_t>(rows, v3d::kNormMaxParts) * (size_t)C * 2 * sizeof(float);
}

int v3d_layer_norm_bwd(const void* grad, const void* feats, const void* residual, const void* weight, const float* mean,
                       const float* rstd, void* grad_feats, void* grad_weight, void* grad_bias, int dtype,
                       int weight_dtype, int64_t rows, int64_t C, void* workspace, size_t workspace_bytes, int device,
                       void* stream) {
  using namespace v3d;
  const char* what = "layer_norm_backward";
  int rc = norm_check(what, dtype, weight_dtype, rows, C, 0.f);
  if (rc != 0) return rc;
  V3D_REQUIRE(rows >= 1, what, "needs at least one row");
  V3D_REQUIRE(grad && feats && mean && rstd, what, "null pointer");
  DeviceGuard guard(device);
  if (guard.rc != 0) return guard.rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  NormArgs a{feats, residual, weight, nullptr, grad, grad_feats, const_cast<float*>(mean), const_cast<float*>(rstd),
             nullptr, rows, (int)C, 0.f};
  Scratch ws;
  if (grad_weight != nullptr || grad_bias != nullptr) {
    rc = ws.acquire(what, workspace, workspace_bytes, v3d_layer_norm_bwd_workspace_bytes(rows, C), s);
    if (rc != 0) return rc;
    a.partial = reinterpret_cast<float*>(ws.base);
  }
  rc = norm_run(a, dtype, weight_dtype, true, grad_weight, grad_bias, s, what);
  return ws.release(what, rc);
}

}  // extern "C"
