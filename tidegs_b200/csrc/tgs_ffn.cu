// Gated feed-forward block over the rows of per-Gaussian features, forward
// and backward:
//   G = X Wg^T, U = X Wu^T, H = silu(G) * U, Y = H Wd^T,
// and with dH = dY Wd, dU = dH silu(G), dG = dH U silu'(G):
//   dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X, dWd = dY^T H.
// The hidden values stay on chip: the backward recomputes G and U.
//
// This file: the entry points, and 32-bit tensors: products on the ordinary
// fp32 pipes, a tile of rows per block, the hidden width in chunks of 32.
// bf16 tensors take the tensor cores (tgs_ffn_tc.cu).
#include "tgs_ffn.cuh"

namespace tgs {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 32;   // rows per tile
constexpr int kHid = 32;    // hidden values per chunk
constexpr int kMaxD = 256;  // also the largest O
constexpr int kMaxH = 4096;

__device__ __forceinline__ float silu_sigmoid(float g) { return 1.f / (1.f + __expf(-g)); }

// Stages rows [r0, r0 + rows) x cols of a row-major matrix as floats with row
// stride ld, zero-filled to `rows`.
template <class T>
__device__ __forceinline__ void stage(float* dst, int ld, const T* src, int64_t stride, int64_t r0,
                                      int rows, int64_t n, int cols) {
  for (int e = threadIdx.x; e < rows * cols; e += kThreads) {
    const int r = e / cols, c = e - r * cols;
    dst[r * ld + c] = r0 + r < n ? to_f32(src[(r0 + r) * stride + c]) : 0.f;
  }
}

// The chunk's hidden values of the tile: thread -> column threadIdx.x % 32,
// rows threadIdx.x / 32 + 8 i.
template <bool kBwd>
__device__ __forceinline__ void hidden(const float* xs, const float* ys, const float* wg,
                                       const float* wu, const float* wd, int ldd, int ldo, int d,
                                       int o, float (&a)[4], float (&b)[4], float (&h)[4]) {
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  float g[4] = {}, u[4] = {}, dh[4] = {};
  for (int k = 0; k < d; ++k) {
    const float wgk = wg[col * ldd + k], wuk = wu[col * ldd + k];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = xs[(row + 8 * i) * ldd + k];
      g[i] += x * wgk;
      u[i] += x * wuk;
    }
  }
  if constexpr (kBwd) {
    for (int k = 0; k < o; ++k) {
      const float wdk = wd[col * ldo + k];
#pragma unroll
      for (int i = 0; i < 4; ++i) dh[i] += ys[(row + 8 * i) * ldo + k] * wdk;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = silu_sigmoid(g[i]), act = g[i] * s;
    h[i] = act * u[i];
    if constexpr (kBwd) {
      a[i] = dh[i] * u[i] * s * (1.f + g[i] * (1.f - s));  // dG
      b[i] = dh[i] * act;                                  // dU
    }
  }
}

template <class T>
__device__ __forceinline__ void stage_chunk(const FfnParams& p, int h0, float* wg, float* wu,
                                            float* wd, int ldd, int ldo) {
  stage(wg, ldd, static_cast<const T*>(p.wg), p.d, h0, kHid, p.h, p.d);
  stage(wu, ldd, static_cast<const T*>(p.wu), p.d, h0, kHid, p.h, p.d);
  const T* src = static_cast<const T*>(p.wd);  // [o, h] -> [hidden, o]
  for (int e = threadIdx.x; e < kHid * p.o; e += kThreads) {
    const int r = e / kHid, c = e - r * kHid;
    wd[c * ldo + r] = h0 + c < p.h ? to_f32(src[static_cast<int64_t>(r) * p.h + h0 + c]) : 0.f;
  }
}

// Forward (Y) or backward (dX): one tile of rows per block, all of H.
template <class T, bool kBwd, int kCols>
__global__ void __launch_bounds__(kThreads) ffn_rows_kernel(const FfnParams p) {
  extern __shared__ float sm[];
  const int ldd = p.d | 1, ldo = p.o | 1;
  float* xs = sm;
  float* wg = xs + kRows * ldd;
  float* wu = wg + kHid * ldd;
  float* wd = wu + kHid * ldd;
  float* hs = wd + kHid * ldo;  // one or two [kRows][33]
  float* ys = hs + 2 * kRows * 33;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows;
  stage(xs, ldd, static_cast<const T*>(p.x), p.x_stride, r0, kRows, p.n, p.d);
  if constexpr (kBwd) stage(ys, ldo, static_cast<const T*>(p.dy), p.dy_stride, r0, kRows, p.n, p.o);
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int out = kBwd ? p.d : p.o;
  float acc[kCols][4] = {};
  for (int h0 = 0; h0 < p.h; h0 += kHid) {
    __syncthreads();
    stage_chunk<T>(p, h0, wg, wu, wd, ldd, ldo);
    __syncthreads();
    float a[4], b[4], h[4];
    hidden<kBwd>(xs, ys, wg, wu, wd, ldd, ldo, p.d, p.o, a, b, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hs[(row + 8 * i) * 33 + col] = kBwd ? a[i] : h[i];
      if constexpr (kBwd) hs[(kRows + row + 8 * i) * 33 + col] = b[i];
    }
    __syncthreads();
    for (int k = 0; k < kHid; ++k) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int c = col + 32 * j;
        if (c < out) {
          const float w0 = kBwd ? wg[k * ldd + c] : wd[k * ldo + c];
          const float w1 = kBwd ? wu[k * ldd + c] : 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[j][i] += hs[(row + 8 * i) * 33 + k] * w0;
            if constexpr (kBwd) acc[j][i] += hs[(kRows + row + 8 * i) * 33 + k] * w1;
          }
        }
      }
    }
  }
  T* y = static_cast<T*>(p.y);
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + row + 8 * i;
      const int c = col + 32 * j;
      if (r < p.n && c < out) y[r * out + c] = from_f32<T>(acc[j][i]);
    }
  }
}

// Weights' gradients of one chunk of H (blockIdx.x) over one slice of the
// rows (blockIdx.y): partial[slice][dWg [H, D] | dWu [H, D] | dWd^T [H, O]].
template <class T, int kCols>
__global__ void __launch_bounds__(kThreads) ffn_weights_kernel(const FfnParams p) {
  extern __shared__ float sm[];
  const int ldd = p.d | 1, ldo = p.o | 1;
  float* xs = sm;
  float* wg = xs + kRows * ldd;
  float* wu = wg + kHid * ldd;
  float* wd = wu + kHid * ldd;
  float* hs = wd + kHid * ldo;  // three [kRows][33]
  float* ys = hs + 3 * kRows * 33;
  const int h0 = blockIdx.x * kHid;
  stage_chunk<T>(p, h0, wg, wu, wd, ldd, ldo);
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int hid = threadIdx.x >> 3, lane = threadIdx.x & 7;
  float ag[kCols] = {}, au[kCols] = {}, ad[kCols] = {};
  for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * kRows; r0 < p.n;
       r0 += static_cast<int64_t>(gridDim.y) * kRows) {
    __syncthreads();
    stage(xs, ldd, static_cast<const T*>(p.x), p.x_stride, r0, kRows, p.n, p.d);
    stage(ys, ldo, static_cast<const T*>(p.dy), p.dy_stride, r0, kRows, p.n, p.o);
    __syncthreads();
    float a[4], b[4], h[4];
    hidden<true>(xs, ys, wg, wu, wd, ldd, ldo, p.d, p.o, a, b, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hs[(row + 8 * i) * 33 + col] = a[i];
      hs[(kRows + row + 8 * i) * 33 + col] = b[i];
      hs[(2 * kRows + row + 8 * i) * 33 + col] = h[i];
    }
    __syncthreads();
    for (int r = 0; r < kRows; ++r) {
      const float dg = hs[r * 33 + hid], du = hs[(kRows + r) * 33 + hid],
                  hh = hs[(2 * kRows + r) * 33 + hid];
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int c = lane + 8 * j;
        const float xv = c < p.d ? xs[r * ldd + c] : 0.f, yv = c < p.o ? ys[r * ldo + c] : 0.f;
        ag[j] += dg * xv;
        au[j] += du * xv;
        ad[j] += hh * yv;
      }
    }
  }
  if (h0 + hid >= p.h) return;
  const int64_t hd = static_cast<int64_t>(p.h) * p.d;
  float* out = p.scratch + blockIdx.y * (2 * hd + static_cast<int64_t>(p.h) * p.o);
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    const int c = lane + 8 * j;
    if (c < p.d) {
      out[static_cast<int64_t>(h0 + hid) * p.d + c] = ag[j];
      out[hd + static_cast<int64_t>(h0 + hid) * p.d + c] = au[j];
    }
    if (c < p.o) out[2 * hd + static_cast<int64_t>(h0 + hid) * p.o + c] = ad[j];
  }
}

// Sums the slices in order and writes the gradients in the weights' layouts.
template <class T>
__global__ void __launch_bounds__(kThreads) ffn_weights_sum_kernel(const float* partial, int slices,
                                                                   int d, int h, int o, T* dwg,
                                                                   T* dwu, T* dwd) {
  const int64_t hd = static_cast<int64_t>(h) * d, ho = static_cast<int64_t>(h) * o;
  const int64_t all = 2 * hd + ho;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (e >= all) return;
  float sum = 0.f;
  for (int s = 0; s < slices; ++s) sum += partial[s * all + e];
  const T v = from_f32<T>(sum);
  if (e < hd) {
    dwg[e] = v;
  } else if (e < 2 * hd) {
    dwu[e - hd] = v;
  } else {
    const int64_t i = (e - 2 * hd) / o, j = (e - 2 * hd) - i * o;
    dwd[j * h + i] = v;
  }
}

int ffn_slices(int64_t n, int h) {
  const int64_t chunks = ceil_div(h, kHid);
  return static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(ceil_div<int64_t>(n, kRows), ceil_div<int64_t>(2 * sm_count(), chunks))));
}

template <class T, bool kBwd, int kCols>
int launch_rows(const FfnParams& p, cudaStream_t s) {
  const int ldd = p.d | 1, ldo = p.o | 1;
  const int smem = 4 * (kRows * ldd + 2 * kHid * ldd + kHid * ldo + 2 * kRows * 33 +
                        (kBwd ? kRows * ldo : 0));
  TGS_CUDA(cudaFuncSetAttribute(ffn_rows_kernel<T, kBwd, kCols>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  ffn_rows_kernel<T, kBwd, kCols>
      <<<static_cast<unsigned>(ceil_div<int64_t>(p.n, kRows)), kThreads, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

template <class T, int kCols>
int launch_weights(const FfnParams& p, int slices, cudaStream_t s) {
  const int ldd = p.d | 1, ldo = p.o | 1;
  const int smem =
      4 * (kRows * ldd + 2 * kHid * ldd + kHid * ldo + 3 * kRows * 33 + kRows * ldo);
  TGS_CUDA(cudaFuncSetAttribute(ffn_weights_kernel<T, kCols>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const dim3 grid(ceil_div(p.h, kHid), slices);
  ffn_weights_kernel<T, kCols><<<grid, kThreads, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

int64_t weights_floats(int64_t n, int d, int h, int o) {
  return ffn_slices(n, h) * static_cast<int64_t>(h) * (2 * d + o);
}

template <class T>
int ffn_weights(const FfnParams& p, cudaStream_t s) {
  const int slices = ffn_slices(p.n, p.h);
  if (int rc = p.d <= 64 && p.o <= 64 ? launch_weights<T, 8>(p, slices, s)
                                      : launch_weights<T, 32>(p, slices, s))
    return rc;
  const int64_t all = static_cast<int64_t>(p.h) * (2 * p.d + p.o);
  ffn_weights_sum_kernel<T><<<static_cast<unsigned>(ceil_div<int64_t>(all, kThreads)), kThreads, 0, s>>>(
      p.scratch, slices, p.d, p.h, p.o, static_cast<T*>(p.dwg), static_cast<T*>(p.dwu),
      static_cast<T*>(p.dwd));
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

int ffn_backward_f32(const FfnParams& p, cudaStream_t s) {
  if (p.y) {
    if (int rc = p.d <= 64 ? launch_rows<float, true, 2>(p, s) : launch_rows<float, true, 8>(p, s))
      return rc;
  }
  return p.dwg ? ffn_weights<float>(p, s) : TGS_OK;
}

int check_ffn(const TgsFfnArgs* a, const char* who) {
  TGS_CHECK_ARG(a != nullptr, "%s: args is NULL", who);
  TGS_CHECK_ARG(a->n >= 0 && a->n <= (1ll << 31) && a->d >= 1 && a->d <= kMaxD && a->o >= 1 &&
                    a->o <= kMaxD && a->h >= 1 && a->h <= kMaxH,
                "%s: bad sizes (n %lld, d %d, h %d, o %d)", who, static_cast<long long>(a->n), a->d,
                a->h, a->o);
  TGS_CHECK_ARG(a->dtype == TGS_F32 || a->dtype == TGS_BF16, "%s: unknown type", who);
  TGS_CHECK_ARG(a->w_gate && a->w_up && a->w_down, "%s: NULL pointer", who);
  TGS_CHECK_ARG(a->n == 0 || a->x, "%s: NULL pointer", who);
  TGS_CHECK_ARG(a->n <= 1 || a->x_stride >= a->d, "%s: rows overlap (stride %lld, d %d)", who,
                static_cast<long long>(a->x_stride), a->d);
  return TGS_OK;
}

FfnParams ffn_params(const TgsFfnArgs& a) {
  FfnParams p{};
  p.x = a.x, p.wg = a.w_gate, p.wu = a.w_up, p.wd = a.w_down, p.y = a.y;
  p.scratch = a.scratch, p.err = a.err;
  p.n = a.n, p.x_stride = a.x_stride, p.d = a.d, p.h = a.h, p.o = a.o;
  return p;
}

}  // namespace
}  // namespace tgs

using namespace tgs;

extern "C" int64_t tgs_ffn_scratch_floats(int64_t n, int32_t d, int32_t h, int32_t o, int32_t dtype,
                                          int32_t backward) {
  if (n <= 0 || d <= 0 || h <= 0 || o <= 0) return 0;
  if (dtype != TGS_F32) return ffn_tc_scratch_floats(n, d, h, o, backward != 0);
  if (!backward) return 0;
  return weights_floats(n, d, h, o);
}

extern "C" int tgs_ffn_fwd(const TgsFfnArgs* a, void* stream) {
  if (int rc = check_ffn(a, "tgs_ffn_fwd")) return rc;
  if (a->n == 0) return TGS_OK;
  TGS_CHECK_ARG(a->y != nullptr, "tgs_ffn_fwd: NULL pointer");
  TGS_CHECK_ARG(a->scratch || !tgs_ffn_scratch_floats(a->n, a->d, a->h, a->o, a->dtype, 0),
                "tgs_ffn_fwd: scratch is NULL");
  const FfnParams p = ffn_params(*a);
  cudaStream_t s = as_stream(stream);
  if (a->dtype == TGS_BF16) return ffn_tc_forward(p, s);
  return p.o <= 64 ? launch_rows<float, false, 2>(p, s) : launch_rows<float, false, 8>(p, s);
}

extern "C" int tgs_ffn_bwd(const TgsFfnBwdArgs* b, void* stream) {
  TGS_CHECK_ARG(b != nullptr, "tgs_ffn_bwd: args is NULL");
  const TgsFfnArgs& a = b->fwd;
  if (int rc = check_ffn(&a, "tgs_ffn_bwd")) return rc;
  const bool weights = b->v_w_gate || b->v_w_up || b->v_w_down;
  TGS_CHECK_ARG(!weights || (b->v_w_gate && b->v_w_up && b->v_w_down),
                "tgs_ffn_bwd: the weights' gradients are all given or none");
  TGS_CHECK_ARG(a.n == 0 || (b->v_y && (b->v_x || weights)), "tgs_ffn_bwd: NULL pointer");
  TGS_CHECK_ARG(a.n <= 1 || b->v_y_stride >= a.o, "tgs_ffn_bwd: rows of v_y overlap");
  TGS_CHECK_ARG(a.scratch || !tgs_ffn_scratch_floats(a.n, a.d, a.h, a.o, a.dtype, 1),
                "tgs_ffn_bwd: scratch is NULL");
  FfnParams p = ffn_params(a);
  p.dy = b->v_y, p.dy_stride = b->v_y_stride, p.y = b->v_x;
  p.dwg = b->v_w_gate, p.dwu = b->v_w_up, p.dwd = b->v_w_down;
  cudaStream_t s = as_stream(stream);
  if (a.n == 0) {
    if (!weights) return TGS_OK;
    const size_t size = a.dtype == TGS_F32 ? 4 : 2, hd = size * a.h * a.d, ho = size * a.h * a.o;
    TGS_CUDA(cudaMemsetAsync(p.dwg, 0, hd, s));
    TGS_CUDA(cudaMemsetAsync(p.dwu, 0, hd, s));
    TGS_CUDA(cudaMemsetAsync(p.dwd, 0, ho, s));
    return TGS_OK;
  }
  return a.dtype == TGS_F32 ? ffn_backward_f32(p, s) : ffn_tc_backward(p, s);
}
