// Layer norm and RMS norm over the last dimension, forward and backward.
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^-1/2          (RMS: mean = 0)
//   y    = (x - mean) * rstd * w + b
//   xh = (x - mean) * rstd,  a = dy * w
//   dx = rstd * (a - mean(a) - xh * mean(a * xh))                        (RMS: without mean(a))
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// Statistics, row sums and the column sums are fp32 in a fixed order (no atomics), so
// results do not change from call to call; every output is rounded once.
#include "dora_common.cuh"

namespace dora {
namespace {

constexpr int kT = 256;  // threads of the row kernels

// Sum over the CTA, in every thread; the same tree each time.  `red` holds one value a warp.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x / 32;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < warps; ++w) t += red[w];
  __syncthreads();
  return t;
}

// One CTA a row, any width and alignment; the row is read three times (from L2 after the first).
template <typename TA, typename TW, bool kRms>
__global__ void __launch_bounds__(kT)
ln_fwd_any_kernel(const TA* __restrict__ x, int64_t ldx, const TW* __restrict__ w, const TW* __restrict__ b, float eps,
                  TA* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int64_t cols) {
  __shared__ float red[kT / 32];
  const float inv = 1.0f / float(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TA* xr = x + r * ldx;
    float mu = 0.f;
    if constexpr (!kRms) {
      float s = 0.f;
      for (int64_t c = threadIdx.x; c < cols; c += kT) s += to_f32(xr[c]);
      mu = block_sum(s, red) * inv;
    }
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rs = rsqrtf(block_sum(q, red) * inv + eps);
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      float v = (to_f32(xr[c]) - mu) * rs;
      if (w) v *= to_f32(w[c]);
      if (b) v += to_f32(b[c]);
      y[r * cols + c] = from_f32<TA>(v);
    }
    if (threadIdx.x == 0) {
      if (!kRms && mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <typename TA, typename TW, bool kRms>
__global__ void __launch_bounds__(kT)
ln_bwd_any_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                  const TW* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                  TA* __restrict__ dx, int64_t rows, int64_t cols) {
  __shared__ float red[kT / 32];
  const float inv = 1.0f / float(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const TA *xr = x + r * ldx, *dr = dy + r * lddy;
    const float mu = kRms ? 0.f : mean[r], rs = rstd[r];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float a = __fmul_rn(to_f32(dr[c]), w ? to_f32(w[c]) : 1.0f);
      s0 += a;
      s1 = fmaf(a, (to_f32(xr[c]) - mu) * rs, s1);
    }
    const float c0 = kRms ? 0.f : block_sum(s0, red) * inv;
    const float c1 = block_sum(s1, red) * inv;
    for (int64_t c = threadIdx.x; c < cols; c += kT) {
      const float a = __fmul_rn(to_f32(dr[c]), w ? to_f32(w[c]) : 1.0f);
      const float xh = (to_f32(xr[c]) - mu) * rs;
      dx[r * cols + c] = from_f32<TA>((a - c0 - xh * c1) * rs);
    }
  }
}

// Column sums over one slab of rows: partial[z][0][c] of dy * xh, partial[z][1][c] of dy.
template <typename TA, bool kRms>
__global__ void __launch_bounds__(kT)
ln_col_any_kernel(const TA* __restrict__ dy, int64_t lddy, const TA* __restrict__ x, int64_t ldx,
                  const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ partial,
                  int64_t rows, int64_t cols) {
  const int64_t c = int64_t(blockIdx.x) * kT + threadIdx.x;
  if (c >= cols) return;
  const int64_t z = blockIdx.y, Z = gridDim.y;
  float dw = 0.f, db = 0.f;
  for (int64_t r = rows * z / Z; r < rows * (z + 1) / Z; ++r) {
    const float d = to_f32(dy[r * lddy + c]);
    const float xh = (to_f32(x[r * ldx + c]) - (kRms ? 0.f : mean[r])) * rstd[r];
    dw = fmaf(d, xh, dw);
    db += d;
  }
  partial[(2 * z) * cols + c] = dw;
  partial[(2 * z + 1) * cols + c] = db;
}

template <typename TW>
__global__ void __launch_bounds__(kT)
ln_col_finish_kernel(const float* __restrict__ partial, int Z, TW* __restrict__ dw, TW* __restrict__ db, int64_t cols) {
  const int64_t c = int64_t(blockIdx.x) * kT + threadIdx.x;
  if (c >= cols) return;
  float a = 0.f, b = 0.f;
  for (int64_t z = 0; z < Z; ++z) {
    a += partial[(2 * z) * cols + c];
    b += partial[(2 * z + 1) * cols + c];
  }
  if (dw) dw[c] = from_f32<TW>(a);
  if (db) db[c] = from_f32<TW>(b);
}

unsigned row_grid(int64_t rows) { return unsigned(rows < (1 << 20) ? rows : (1 << 20)); }

int col_slabs(int64_t rows, int64_t cols) {
  const int64_t tiles = (cols + kT - 1) / kT;
  int64_t z = (int64_t(num_sms()) * 8 + tiles - 1) / tiles;
  if (z > rows) z = rows;
  return int(z < 1 ? 1 : z > 1024 ? 1024 : z);
}

template <typename TA, typename TW, bool kRms>
int launch_fwd(const void* x, int64_t ldx, const void* w, const void* b, float eps, void* y, float* mean, float* rstd,
               int64_t rows, int64_t cols, cudaStream_t st) {
  ln_fwd_any_kernel<TA, TW, kRms><<<row_grid(rows), kT, 0, st>>>(
      static_cast<const TA*>(x), ldx, static_cast<const TW*>(w), static_cast<const TW*>(b), eps, static_cast<TA*>(y),
      mean, rstd, rows, cols);
  return check_launch();
}

template <typename TA, typename TW, bool kRms>
int launch_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const float* mean,
               const float* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, int64_t rows, int64_t cols,
               cudaStream_t st) {
  auto D = static_cast<const TA*>(dy);
  auto X = static_cast<const TA*>(x);
  const int Z = col_slabs(rows, cols);
  if ((dw || db) && (!ws || ws_bytes < size_t(Z) * 2 * size_t(cols) * 4 || (reinterpret_cast<uintptr_t>(ws) & 15u)))
    return DORA_ERR_WORKSPACE;
  if (dx && rows) {
    ln_bwd_any_kernel<TA, TW, kRms><<<row_grid(rows), kT, 0, st>>>(D, lddy, X, ldx, static_cast<const TW*>(w), mean,
                                                                   rstd, static_cast<TA*>(dx), rows, cols);
    const int e = check_launch();
    if (e) return e;
  }
  if (!dw && !db) return DORA_OK;
  const unsigned tiles = unsigned((cols + kT - 1) / kT);
  auto part = static_cast<float*>(ws);
  ln_col_any_kernel<TA, kRms><<<dim3(tiles, unsigned(Z)), kT, 0, st>>>(D, lddy, X, ldx, mean, rstd, part, rows, cols);
  const int e = check_launch();
  if (e) return e;
  ln_col_finish_kernel<TW><<<tiles, kT, 0, st>>>(part, Z, static_cast<TW*>(dw), static_cast<TW*>(db), cols);
  return check_launch();
}

bool shape_ok(int64_t rows, int64_t cols, int64_t ld) {
  return rows >= 0 && cols >= 0 && ld >= cols && cols <= (int64_t(1) << 30) && rows <= (int64_t(1) << 40);
}
bool types_ok(int act_dtype, int w_dtype) {
  return dtype_ok(act_dtype) && (w_dtype == act_dtype || w_dtype == DORA_DTYPE_F32);
}

template <bool kRms, typename F>
int by_type(int act_dtype, int w_dtype, F f) {
  switch (act_dtype) {
    case DORA_DTYPE_BF16:
      return w_dtype == DORA_DTYPE_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
    case DORA_DTYPE_F16: return w_dtype == DORA_DTYPE_F32 ? f(__half(), float()) : f(__half(), __half());
    default: return f(float(), float());
  }
}

template <bool kRms>
int norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int w_dtype, double eps, void* y, void* mean,
             void* rstd, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  if (!shape_ok(rows, cols, ldx) || !types_ok(act_dtype, w_dtype) || !(eps >= 0)) return DORA_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return DORA_OK;
  if (!x || !y || x == y) return DORA_ERR_INVALID_ARGUMENT;
  return by_type<kRms>(act_dtype, w_dtype, [&](auto ta, auto tw) {
    return launch_fwd<decltype(ta), decltype(tw), kRms>(x, ldx, w, b, float(eps), y, static_cast<float*>(mean),
                                                        static_cast<float*>(rstd), rows, cols,
                                                        static_cast<cudaStream_t>(stream));
  });
}

template <bool kRms>
int norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int w_dtype, const void* mean,
             const void* rstd, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, int64_t rows, int64_t cols,
             int act_dtype, void* stream) {
  if (!shape_ok(rows, cols, ldx) || lddy < cols || !types_ok(act_dtype, w_dtype)) return DORA_ERR_INVALID_ARGUMENT;
  if (cols == 0 || (!dx && !dw && !db)) return DORA_OK;
  if (rows && (!dy || !x || !rstd || (!kRms && !mean) || (dx && (dx == dy || dx == x)))) return DORA_ERR_INVALID_ARGUMENT;
  if (rows == 0 && !dw && !db) return DORA_OK;
  return by_type<kRms>(act_dtype, w_dtype, [&](auto ta, auto tw) {
    return launch_bwd<decltype(ta), decltype(tw), kRms>(dy, lddy, x, ldx, w, static_cast<const float*>(mean),
                                                        static_cast<const float*>(rstd), dx, dw, db, ws, ws_bytes, rows,
                                                        cols, static_cast<cudaStream_t>(stream));
  });
}

}  // namespace
}  // namespace dora

using namespace dora;

extern "C" int dora_layer_norm_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, int w_dtype,
                                   double eps, void* y, void* mean, void* rstd, int64_t rows, int64_t cols,
                                   int act_dtype, void* stream) {
  return norm_fwd<false>(x, ldx, weight, bias, w_dtype, eps, y, mean, rstd, rows, cols, act_dtype, stream);
}

extern "C" int dora_rms_norm_fwd(const void* x, int64_t ldx, const void* weight, int w_dtype, double eps, void* y,
                                 void* rstd, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  return norm_fwd<true>(x, ldx, weight, nullptr, w_dtype, eps, y, nullptr, rstd, rows, cols, act_dtype, stream);
}

extern "C" size_t dora_layer_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (!shape_ok(rows, cols, cols) || cols == 0) return 0;
  return size_t(col_slabs(rows, cols)) * 2 * size_t(cols) * 4;
}

extern "C" int dora_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                   int w_dtype, const void* mean, const void* rstd, void* dx, void* d_weight,
                                   void* d_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols,
                                   int act_dtype, void* stream) {
  return norm_bwd<false>(dy, lddy, x, ldx, weight, w_dtype, mean, rstd, dx, d_weight, d_bias, workspace,
                         workspace_bytes, rows, cols, act_dtype, stream);
}

extern "C" int dora_rms_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                 int w_dtype, const void* rstd, void* dx, void* d_weight, void* workspace,
                                 size_t workspace_bytes, int64_t rows, int64_t cols, int act_dtype, void* stream) {
  return norm_bwd<true>(dy, lddy, x, ldx, weight, w_dtype, nullptr, rstd, dx, d_weight, nullptr, workspace,
                        workspace_bytes, rows, cols, act_dtype, stream);
}
