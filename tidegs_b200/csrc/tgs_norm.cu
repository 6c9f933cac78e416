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
// Bound: HBM. A group of `lanes` threads holds kU rows at a time, as they were
// loaded (16-byte vectors, or single values where width or alignment forbid
// them), so that enough bytes are on their way: a warp or a part of one per
// row, or the whole block for wide rows, where the kU rows share the barriers.
// Measured: 2,097,152 rows of 64 bf16, forward 104 us (5.2 TB/s, 80 % of the
// copy rate), backward 197 us; of 64 fp32 186 and 255 us (5.8 and 6.3 TB/s);
// 786,432 rows of 59 fp32, which only take single loads, 83 and 157 us.
#include <atomic>

#include "tgs_common.cuh"
#include "tgs_vec.cuh"

namespace tgs {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxC = 8192;
constexpr int kNormBlocksPerSm = 8;

// Sums of kU values over the group of threads that holds a row: `lanes`
// neighbours within a warp, or the whole block (kBlock) through shared memory.
template <bool kBlock, int kU>
__device__ __forceinline__ void group_sum(float (&v)[kU], int lanes, float (*red)[kU]) {
  if constexpr (kBlock) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < kU; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < kU; ++k) red[threadIdx.x >> 5][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kNormThreads / 32; ++w) v[k] += red[w][k];
    }
  } else {
    for (int off = lanes >> 1; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < kU; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
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

// kVec values per load, kNv loads per thread and row, kU rows at a time:
// thread t of a group holds columns (t + lanes j) kVec + i.
template <class T, int kVec, int kNv, int kU, bool kBlock>
struct NormRows {
  Packed<T, kVec> x[kU][kNv];

  __device__ __forceinline__ void load(const T* src, int64_t stride, int64_t r0, int64_t n,
                                       int groups, int t, int lanes, int c) {
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int64_t r = r0 + static_cast<int64_t>(k) * groups;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (t + lanes * j) * kVec;
        x[k][j].load(src + r * stride + col, r < n && col < c);
      }
    }
  }

  // Means, and 1 / sqrt(variance + eps), of the rows.
  __device__ __forceinline__ void stats(float (&mean)[kU], float (&rstd)[kU], int t, int lanes, int c,
                                        float inv_c, float eps, float (*red)[kU]) {
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      mean[k] = 0.f;
#pragma unroll
      for (int j = 0; j < kNv; ++j)
#pragma unroll
        for (int i = 0; i < kVec; ++i) mean[k] += x[k][j].get(i);
    }
    group_sum<kBlock>(mean, lanes, red);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      mean[k] *= inv_c;
      rstd[k] = 0.f;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const bool in = (t + lanes * j) * kVec < c;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float d = in ? x[k][j].get(i) - mean[k] : 0.f;
          rstd[k] += d * d;
        }
      }
    }
    group_sum<kBlock>(rstd, lanes, red);
#pragma unroll
    for (int k = 0; k < kU; ++k) rstd[k] = rsqrtf(rstd[k] * inv_c + eps);
  }
};

template <class T, int kVec, int kNv, int kU, bool kBlock>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_kernel(const NormParams p) {
  __shared__ float red[kNormThreads / 32][kU];
  const int lanes = p.lanes, c = p.c;
  const int t = threadIdx.x & (lanes - 1);
  const int groups = kNormThreads / lanes;
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
  T* y = static_cast<T*>(p.y);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups * kU; base < p.n;
       base += static_cast<int64_t>(gridDim.x) * groups * kU) {
    const int64_t r0 = base + threadIdx.x / lanes;
    NormRows<T, kVec, kNv, kU, kBlock> rows;
    rows.load(static_cast<const T*>(p.x), p.x_stride, r0, p.n, groups, t, lanes, c);
    float mean[kU], rstd[kU];
    rows.stats(mean, rstd, t, lanes, c, inv_c, p.eps, red);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int64_t r = r0 + static_cast<int64_t>(k) * groups;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (t + lanes * j) * kVec;
        if (r < p.n && col < c) {
          float o[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            o[i] = (rows.x[k][j].get(i) - mean[k]) * rstd[k] * w[j][i] + b[j][i];
          store_vec<T, kVec>(y + r * c + col, o);
        }
      }
    }
  }
}

// Blocks to an SM that the compiler has to leave registers for (0: it chooses).
// Rows of many values to a thread are held back by too few of them. 200 MB in
// each tensor, us with this rule and with its own choice, by type and columns:
//   16 values, two blocks: bf16 64, 256, 512 as they were (155, 168, 177); single
//      loads, fp32 257, 301, 511 329, 298, 235 (436, 394, 292), bf16 301, 509
//      690, 480 (873, 557)
//   24 values, two: bf16 520, 640, 768 233, 196, 171 (320, 271, 232)
//   32 values, one: bf16 1024 206 (238); two blocks 348
// Fewer values, and rows that a block shares, have registers for more anyway.
constexpr int norm_min_blocks(int values, bool block) {
  return block || values < 16 ? 0 : values <= 24 ? 2 : 1;
}

template <class T, int kVec, int kNv, int kU, bool kBlock>
__global__ void __launch_bounds__(kNormThreads, norm_min_blocks(kVec * kNv, kBlock)) norm_bwd_kernel(const NormParams p) {
  extern __shared__ float acc[];  // [2, C]: the block's parameter gradients
  __shared__ float red[kNormThreads / 32][kU];
  const int lanes = p.lanes, c = p.c;
  const int t = threadIdx.x & (lanes - 1);
  const int groups = kNormThreads / lanes;
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
  T* dx = static_cast<T*>(p.y);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups * kU; base < p.n;
       base += static_cast<int64_t>(gridDim.x) * groups * kU) {
    const int64_t r0 = base + threadIdx.x / lanes;
    NormRows<T, kVec, kNv, kU, kBlock> rows, grads;
    rows.load(static_cast<const T*>(p.x), p.x_stride, r0, p.n, groups, t, lanes, c);
    grads.load(static_cast<const T*>(p.dy), p.dy_stride, r0, p.n, groups, t, lanes, c);
    float mean[kU], rstd[kU], s1[kU], s2[kU];
    rows.stats(mean, rstd, t, lanes, c, inv_c, p.eps, red);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      s1[k] = s2[k] = 0.f;
      if (r0 + static_cast<int64_t>(k) * groups < p.n) {  // rows past the end add nothing
#pragma unroll
        for (int j = 0; j < kNv; ++j) {
          if ((t + lanes * j) * kVec < c) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
              const float z = (rows.x[k][j].get(i) - mean[k]) * rstd[k], g = grads.x[k][j].get(i);
              db[j][i] += g;
              dw[j][i] += g * z;
              s1[k] += g * w[j][i];
              s2[k] += g * w[j][i] * z;
            }
          }
        }
      }
    }
    group_sum<kBlock>(s1, lanes, red);
    group_sum<kBlock>(s2, lanes, red);
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int64_t r = r0 + static_cast<int64_t>(k) * groups;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (t + lanes * j) * kVec;
        if (r < p.n && col < c && dx) {
          float o[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const float z = (rows.x[k][j].get(i) - mean[k]) * rstd[k];
            o[i] = rstd[k] * (grads.x[k][j].get(i) * w[j][i] - s1[k] * inv_c - z * (s2[k] * inv_c));
          }
          store_vec<T, kVec>(dx + r * c + col, o);
        }
      }
    }
  }
  if (p.partial == nullptr) return;
  // The block's groups add their sums one after another, so the order of the
  // additions is fixed; within a warp, by exchanges.
  const int per_warp = lanes < 32 ? 32 / lanes : 1;
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      for (int off = lanes; off < 32; off <<= 1) {
        dw[j][i] += __shfl_xor_sync(0xffffffffu, dw[j][i], off);
        db[j][i] += __shfl_xor_sync(0xffffffffu, db[j][i], off);
      }
    }
  }
  const int turns = groups / per_warp, mine = threadIdx.x / lanes;
  for (int turn = 0; turn < turns; ++turn) {
    __syncthreads();
    if (mine == turn * per_warp) {
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

// Column sums of the blocks' partial gradients: 32 columns per block, 32
// threads per column.
__global__ void __launch_bounds__(1024) norm_param_kernel(const float* __restrict__ partial,
                                                          int blocks, int c, int dtype,
                                                          void* dweight, void* dbias) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (e < 2 * c) {
#pragma unroll 4
    for (int b = k; b < blocks; b += 32) sum += partial[static_cast<int64_t>(b) * 2 * c + e];
  }
  s[k][lane] = sum;
  __syncthreads();
  // column k of the block's 32: its 32 partial sums, added as a tree
  sum = s[lane][k];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const int col = blockIdx.x * 32 + k;
  if (lane != 0 || col >= 2 * c) return;
  if (col < c) {
    if (dweight) store_param(dweight, dtype, col, sum);
  } else if (dbias) {
    store_param(dbias, dtype, col - c, sum);
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

// Threads per row: the fewest neighbours (a power of two) that hold it with
// kNv loads each.
int norm_lanes(int c, int per_thread) {
  int lanes = 1;
  while (lanes < kNormThreads && lanes * per_thread < c) lanes *= 2;
  return lanes;
}

template <class T, int kVec, int kNv, int kU, bool kBlock, bool kBwd>
int launch_norm(NormParams p, cudaStream_t s, int* blocks) {
  const auto kernel = kBwd ? norm_bwd_kernel<T, kVec, kNv, kU, kBlock>
                           : norm_fwd_kernel<T, kVec, kNv, kU, kBlock>;
  p.lanes = kBlock ? kNormThreads : norm_lanes(p.c, kVec * kNv);
  const int64_t rows = static_cast<int64_t>(kNormThreads / p.lanes) * kU;
  const int smem = kBwd && p.partial ? 2 * p.c * static_cast<int>(sizeof(float)) : 0;
  // The default limit, 48 KB, covers the kernel's own arrays too. One limit for
  // every width: it belongs to the kernel, and another thread may be launching it.
  constexpr int kMostSmem = 2 * kNormMaxC * static_cast<int>(sizeof(float));
  if (smem > 32 * 1024)
    TGS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
  // As many blocks as are resident at once: each sums its parameter gradients
  // and hands them over once.
  static std::atomic<int> known{0};
  int resident = known.load(std::memory_order_relaxed);
  if (resident == 0) {
    int n = 0;
    TGS_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kNormThreads, 0));
    resident = std::max(1, std::min(n, kNormBlocksPerSm));
    known.store(resident, std::memory_order_relaxed);
  }
  *blocks = static_cast<int>(std::min<int64_t>(ceil_div<int64_t>(p.n, rows),
                                               static_cast<int64_t>(sm_count()) * resident));
  kernel<<<*blocks, kNormThreads, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

// kNv and kU: few threads to a row, for few exchanges (at 59 columns of fp32,
// 8 threads of 8 values against 32 of 2), while a thread keeps about 64 bytes
// of each of its tensors on their way and no more values than its registers
// hold (the backward has four sets). Three vectors a thread, of a warp to the row,
// against four: bf16 520, 640 and 768 columns backward 233, 196 and 171 us of
// 334, 281 and 240, fp32 260, 320 and 384 146, 127 and 113 of 169, 145 and 129,
// forward 78, 69 and 68 of 87, 79 and 72 (200 MB in each tensor).
template <class T, int kVec, bool kBwd>
int launch_norm_vec(const NormParams& p, cudaStream_t s, int* blocks) {
  constexpr int kWarp = 32 * kVec, kWide = kNormThreads * kVec;  // values of one load
  const int c = p.c;
  if constexpr (kVec == 1) {
    if (c <= 4) return launch_norm<T, kVec, 4, kBwd ? 2 : 4, false, kBwd>(p, s, blocks);
    if (c <= 8 * kWarp) return launch_norm<T, kVec, 8, kBwd ? 1 : 2, false, kBwd>(p, s, blocks);
    if (c <= 16 * kWarp) return launch_norm<T, kVec, 16, 1, false, kBwd>(p, s, blocks);
    if (c <= 4 * kWide) return launch_norm<T, kVec, 4, 2, true, kBwd>(p, s, blocks);
    return launch_norm<T, kVec, 32, 1, true, kBwd>(p, s, blocks);
  } else {
    if (c <= 4 * kVec) return launch_norm<T, kVec, 1, kBwd ? 2 : 4, false, kBwd>(p, s, blocks);
    if (c <= 2 * kWarp) return launch_norm<T, kVec, 2, kBwd ? 1 : 2, false, kBwd>(p, s, blocks);
    if (c <= 3 * kWarp) return launch_norm<T, kVec, 3, 1, false, kBwd>(p, s, blocks);
    if (c <= 4 * kWarp) return launch_norm<T, kVec, 4, 1, false, kBwd>(p, s, blocks);
    if (c <= kWide) return launch_norm<T, kVec, 1, 4, true, kBwd>(p, s, blocks);
    if (c <= 2 * kWide) return launch_norm<T, kVec, 2, 2, true, kBwd>(p, s, blocks);
    return launch_norm<T, kVec, kNormMaxC / kWide, 1, true, kBwd>(p, s, blocks);
  }
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
  return std::min<int64_t>(n, static_cast<int64_t>(sm_count()) * kNormBlocksPerSm) * 2 * c;
}

extern "C" int tgs_layer_norm_bwd(const TgsLayerNormBwdArgs* b, void* stream) {
  launches() = 0;
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
    norm_param_kernel<<<ceil_div(2 * a.c, 32), 1024, 0, s>>>(b->scratch, blocks, a.c, a.param_dtype,
                                                           b->v_weight, b->v_bias);
    TGS_LAUNCH_CHECK();
  }
  return TGS_OK;
}
