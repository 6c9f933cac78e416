// Layer norm over the rows of per-Gaussian features, forward and backward.
//
// Forward, for a row x of C values: m = mean(x), s = 1 / sqrt(mean((x - m)^2)
// + eps), z = (x - m) s, y = z w + b. Backward, with v = dy w:
//   dx = s (v - mean(v) - z mean(v z)),  dw = sum_rows dy z,  db = sum_rows dy.
// A row is loaded once and stays in registers, so the mean is taken before
// the squares (no cancellation) and the backward recomputes the statistics
// from the row it reads anyway instead of reading them back. All sums are in
// 32 bits; only y and the gradients are rounded to the tensors' types, once.
//
// Bound: HBM. A group of `lanes` threads (a power of two, at most a warp)
// holds one row of at most 1024 values; wider rows take a whole block.
#include "tgs_common.cuh"
#include "tgs_vec.cuh"

namespace tgs {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxC = 8192;

// Sum over the group of threads that holds a row: `lanes` neighbours within a
// warp, or the whole block (kBlock) through shared memory.
template <bool kBlock>
__device__ __forceinline__ float group_sum(float v, int lanes, float* red) {
  if constexpr (kBlock) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) t += red[w];
    return t;
  } else {
    for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  }
}

struct NormParams {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;   // dx in the backward
  float* partial;  // [blocks, 2, C] (backward with parameter gradients)
  int64_t n, x_stride, dy_stride;
  int c, param_dtype, lanes;
  float eps;
};

// kVec values per load, kNv loads per thread and row: thread t of a group
// holds columns (t + lanes j) kVec + i.
template <class T, int kVec, int kNv, bool kBlock>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_kernel(const NormParams p) {
  __shared__ float red[kNormThreads / 32];
  const int lanes = p.lanes, c = p.c;
  const int t = threadIdx.x & (lanes - 1);
  const int groups = kNormThreads / lanes;
  const int group = threadIdx.x / lanes;
  float w[kNv][kVec], b[kNv][kVec];
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int col = (t + lanes * j) * kVec + i;
      w[j][i] = col < c && p.weight ? load_param(p.weight, p.param_dtype, col) : 1.f;
      b[j][i] = col < c && p.bias ? load_param(p.bias, p.param_dtype, col) : 0.f;
    }
  }
  const float inv_c = 1.f / static_cast<float>(c);
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * groups; r0 < p.n;
       r0 += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t r = r0 + group;
    const bool row = r < p.n;
    float v[kNv][kVec];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (t + lanes * j) * kVec;
      load_vec<T, kVec>(x + r * p.x_stride + col, row && col < c, v[j]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum += v[j][i];
    }
    const float mean = group_sum<kBlock>(sum, lanes, red) * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const bool in = (t + lanes * j) * kVec < c;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[j][i] -= mean;
        sq += in ? v[j][i] * v[j][i] : 0.f;
      }
    }
    const float rstd = rsqrtf(group_sum<kBlock>(sq, lanes, red) * inv_c + p.eps);
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (t + lanes * j) * kVec;
      if (row && col < c) {
        float o[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) o[i] = v[j][i] * rstd * w[j][i] + b[j][i];
        store_vec<T, kVec>(y + r * c + col, o);
      }
    }
  }
}

template <class T, int kVec, int kNv, bool kBlock>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_kernel(const NormParams p) {
  extern __shared__ float acc[];  // [2, C]: the block's parameter gradients
  __shared__ float red[kNormThreads / 32];
  const int lanes = p.lanes, c = p.c;
  const int t = threadIdx.x & (lanes - 1);
  const int groups = kNormThreads / lanes;
  const int group = threadIdx.x / lanes;
  float w[kNv][kVec], dw[kNv][kVec], db[kNv][kVec];
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int col = (t + lanes * j) * kVec + i;
      w[j][i] = col < c && p.weight ? load_param(p.weight, p.param_dtype, col) : 1.f;
      dw[j][i] = db[j][i] = 0.f;
    }
  }
  const float inv_c = 1.f / static_cast<float>(c);
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.y);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * groups; r0 < p.n;
       r0 += static_cast<int64_t>(gridDim.x) * groups) {
    const int64_t r = r0 + group;
    const bool row = r < p.n;
    float v[kNv][kVec], g[kNv][kVec];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (t + lanes * j) * kVec;
      load_vec<T, kVec>(x + r * p.x_stride + col, row && col < c, v[j]);
      load_vec<T, kVec>(dy + r * p.dy_stride + col, row && col < c, g[j]);
    }
#pragma unroll
    for (int j = 0; j < kNv; ++j)
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum += v[j][i];
    const float mean = group_sum<kBlock>(sum, lanes, red) * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const bool in = (t + lanes * j) * kVec < c;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[j][i] = in ? v[j][i] - mean : 0.f;
        sq += v[j][i] * v[j][i];
      }
    }
    const float rstd = rsqrtf(group_sum<kBlock>(sq, lanes, red) * inv_c + p.eps);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[j][i] *= rstd;
        if (row) {  // rows past the end add nothing
          db[j][i] += g[j][i];
          dw[j][i] += g[j][i] * v[j][i];
        }
        g[j][i] *= w[j][i];
        s1 += g[j][i];
        s2 += g[j][i] * v[j][i];
      }
    }
    s1 = group_sum<kBlock>(s1, lanes, red) * inv_c;
    s2 = group_sum<kBlock>(s2, lanes, red) * inv_c;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (t + lanes * j) * kVec;
      if (row && col < c && dx) {
        float o[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) o[i] = rstd * (g[j][i] - s1 - v[j][i] * s2);
        store_vec<T, kVec>(dx + r * c + col, o);
      }
    }
  }
  if (p.partial == nullptr) return;
  // The block's groups add their sums one after another, so the order of the
  // additions is fixed.
  for (int turn = 0; turn < groups; ++turn) {
    __syncthreads();
    if (group == turn) {
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int col = (t + lanes * j) * kVec + i;
          if (col < c) {
            acc[col] = (turn ? acc[col] : 0.f) + dw[j][i];
            acc[c + col] = (turn ? acc[c + col] : 0.f) + db[j][i];
          }
        }
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * c; e += kNormThreads)
    p.partial[static_cast<int64_t>(blockIdx.x) * 2 * c + e] = acc[e];
}

// Column sums of the blocks' partial gradients: 32 columns per block, eight
// threads per column.
__global__ void __launch_bounds__(256) norm_param_kernel(const float* __restrict__ partial,
                                                         int blocks, int c, int dtype,
                                                         void* dweight, void* dbias) {
  __shared__ float s[8][33];
  const int e = blockIdx.x * 32 + (threadIdx.x & 31);
  const int k = threadIdx.x >> 5;
  float sum = 0.f;
  if (e < 2 * c)
    for (int b = k; b < blocks; b += 8) sum += partial[static_cast<int64_t>(b) * 2 * c + e];
  s[k][threadIdx.x & 31] = sum;
  __syncthreads();
  if (k != 0 || e >= 2 * c) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += s[i][threadIdx.x & 31];
  if (e < c) {
    if (dweight) store_param(dweight, dtype, e, sum);
  } else if (dbias) {
    store_param(dbias, dtype, e - c, sum);
  }
}

int check_norm(const TgsLayerNormArgs* a, const char* who) {
  TGS_CHECK_ARG(a != nullptr, "%s: args is NULL", who);
  TGS_CHECK_ARG(a->n >= 0 && a->c >= 1 && a->c <= kNormMaxC, "%s: bad sizes (n %lld, c %d)", who,
                static_cast<long long>(a->n), a->c);
  TGS_CHECK_ARG(valid_dtype(a->dtype) && valid_dtype(a->param_dtype), "%s: unknown type", who);
  TGS_CHECK_ARG(a->n == 0 || a->x, "%s: NULL pointer", who);
  TGS_CHECK_ARG(a->n <= 1 || a->x_stride >= a->c, "%s: rows overlap (stride %lld, c %d)", who,
                static_cast<long long>(a->x_stride), a->c);
  return TGS_OK;
}

int norm_blocks(int64_t n, int lanes) {
  const int64_t groups = kNormThreads / lanes;
  return static_cast<int>(std::min<int64_t>(ceil_div<int64_t>(n, groups),
                                            static_cast<int64_t>(sm_count()) * 8));
}

// Threads per row: the fewest neighbours (a power of two) that hold it with
// kNv loads each.
int norm_lanes(int c, int per_thread) {
  int lanes = 1;
  while (lanes < kNormThreads && lanes * per_thread < c) lanes *= 2;
  return lanes;
}

template <class T, int kVec, int kNv, bool kBlock, bool kBwd>
int launch_norm(NormParams p, cudaStream_t s, int* blocks) {
  p.lanes = kBlock ? kNormThreads : norm_lanes(p.c, kVec * kNv);
  *blocks = norm_blocks(p.n, p.lanes);
  if constexpr (kBwd) {
    const int smem = p.partial ? 2 * p.c * static_cast<int>(sizeof(float)) : 0;
    TGS_CUDA(cudaFuncSetAttribute(norm_bwd_kernel<T, kVec, kNv, kBlock>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    norm_bwd_kernel<T, kVec, kNv, kBlock><<<*blocks, kNormThreads, smem, s>>>(p);
  } else {
    norm_fwd_kernel<T, kVec, kNv, kBlock><<<*blocks, kNormThreads, 0, s>>>(p);
  }
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

template <class T, int kVec, bool kBwd>
int launch_norm_vec(const NormParams& p, cudaStream_t s, int* blocks) {
  constexpr int kWarp = 32 * kVec;  // values that one load of a warp covers
  if (p.c <= kWarp) return launch_norm<T, kVec, 1, false, kBwd>(p, s, blocks);
  if (p.c <= 2 * kWarp) return launch_norm<T, kVec, 2, false, kBwd>(p, s, blocks);
  if (p.c <= 4 * kWarp) return launch_norm<T, kVec, 4, false, kBwd>(p, s, blocks);
  constexpr int kWide = kNormMaxC / (kNormThreads * kVec);
  if (p.c <= kNormThreads * kVec * (kWide / 4 > 0 ? kWide / 4 : 1))
    return launch_norm<T, kVec, (kWide / 4 > 0 ? kWide / 4 : 1), true, kBwd>(p, s, blocks);
  return launch_norm<T, kVec, kWide, true, kBwd>(p, s, blocks);
}

template <class T, bool kBwd>
int launch_norm_type(const NormParams& p, cudaStream_t s, int* blocks) {
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = p.c % kWide == 0 && aligned16(p.x) && p.x_stride % kWide == 0 &&
                    aligned16(p.y) && (!kBwd || (aligned16(p.dy) && p.dy_stride % kWide == 0));
  if (wide) return launch_norm_vec<T, kWide, kBwd>(p, s, blocks);
  return launch_norm_vec<T, 1, kBwd>(p, s, blocks);
}

template <bool kBwd>
int launch_norm_any(const NormParams& p, int dtype, cudaStream_t s, int* blocks) {
  switch (dtype) {
    case TGS_F32: return launch_norm_type<float, kBwd>(p, s, blocks);
    case TGS_BF16: return launch_norm_type<__nv_bfloat16, kBwd>(p, s, blocks);
    default: return launch_norm_type<__half, kBwd>(p, s, blocks);
  }
}

NormParams norm_params(const TgsLayerNormArgs& a) {
  NormParams p{};
  p.x = a.x, p.weight = a.weight, p.bias = a.bias, p.y = a.y;
  p.n = a.n, p.x_stride = a.x_stride, p.c = a.c, p.param_dtype = a.param_dtype, p.eps = a.eps;
  return p;
}

}  // namespace
}  // namespace tgs

using namespace tgs;

extern "C" int tgs_layer_norm_fwd(const TgsLayerNormArgs* a, void* stream) {
  if (int rc = check_norm(a, "tgs_layer_norm_fwd")) return rc;
  if (a->n == 0) return TGS_OK;
  TGS_CHECK_ARG(a->y != nullptr, "tgs_layer_norm_fwd: NULL pointer");
  int blocks = 0;
  return launch_norm_any<false>(norm_params(*a), a->dtype, as_stream(stream), &blocks);
}

extern "C" int64_t tgs_layer_norm_scratch_floats(int64_t n, int32_t c) {
  if (n <= 0 || c <= 0) return 0;
  return std::min<int64_t>(n, static_cast<int64_t>(sm_count()) * 8) * 2 * c;
}

extern "C" int tgs_layer_norm_bwd(const TgsLayerNormBwdArgs* b, void* stream) {
  TGS_CHECK_ARG(b != nullptr, "tgs_layer_norm_bwd: args is NULL");
  const TgsLayerNormArgs& a = b->fwd;
  if (int rc = check_norm(&a, "tgs_layer_norm_bwd")) return rc;
  const bool params = b->v_weight || b->v_bias;
  cudaStream_t s = as_stream(stream);
  int blocks = 0;
  if (a.n > 0) {
    TGS_CHECK_ARG(b->v_y && (b->v_x || params), "tgs_layer_norm_bwd: NULL pointer");
    TGS_CHECK_ARG(a.n <= 1 || b->v_y_stride >= a.c, "tgs_layer_norm_bwd: rows of v_y overlap");
    TGS_CHECK_ARG(!params || b->scratch, "tgs_layer_norm_bwd: scratch is NULL");
    NormParams p = norm_params(a);
    p.dy = b->v_y, p.dy_stride = b->v_y_stride, p.y = b->v_x;
    p.partial = params ? b->scratch : nullptr;
    if (int rc = launch_norm_any<true>(p, a.dtype, s, &blocks)) return rc;
  }
  if (params) {
    norm_param_kernel<<<ceil_div(2 * a.c, 32), 256, 0, s>>>(b->scratch, blocks, a.c, a.param_dtype,
                                                           b->v_weight, b->v_bias);
    TGS_LAUNCH_CHECK();
  }
  return TGS_OK;
}
