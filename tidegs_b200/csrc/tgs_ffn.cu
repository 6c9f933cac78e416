// Gated feed-forward block over the rows of per-Gaussian features, forward
// and backward:
//   G = X Wg^T, U = X Wu^T, H = silu(G) * U, Y = H Wd^T,
// and with dH = dY Wd, dU = dH silu(G), dG = dH U silu'(G):
//   dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X, dWd = dY^T H.
// The hidden values stay on chip: the backward recomputes G and U.
//
// This file: the entry points, and narrow blocks of 32-bit tensors, whose
// products run on the ordinary fp32 pipes. bf16 tensors take the tensor cores
// (tgs_ffn_tc.cu), and wide blocks of 32-bit tensors too (tgs_ffn_tc32.cu).
//
// A block of 256 threads, 16 x 16, works on a tile of 16 kR rows and chunks of
// 32 hidden values. Everything lies in shared memory with the contracted index
// first and neighbouring rows (or hidden values) together, so that a product
// reads 16 bytes at a time, and multiply-adds go in pairs (fma.rn.f32x2): at
// kR = 8, 16 pairs for four 16-byte reads. Bound: the fp32 pipes. 131,071 rows
// of 35 -> 96 -> 3: forward 71 us, backward 417 us.
#include "tgs_ffn.cuh"

namespace tgs {
namespace {

constexpr int kThreads = 256;
constexpr int kHid = 32;    // hidden values per chunk, two per thread column
constexpr int kMaxD = 256;  // also the largest O
constexpr int kMaxH = 4096;
constexpr int kLdW = 2 * kHid + 4;  // row of Wg, Wu: g g u u per pair of hidden values
constexpr int kLdD = kHid + 4;      // row of Wd

__host__ __device__ constexpr int rows_ld(int r) { return 16 * r + 4; }

// 4 bytes global -> shared, or zero where !on; completes with the group. The
// copies transpose, and leave no register waiting for memory.
__device__ __forceinline__ void copy4(float* dst, const float* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src),
               "r"(on ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <int kR>
struct Tile {
  static constexpr int kRows = 16 * kR, kLd = rows_ld(kR);
  const FfnParams& p;
  float* xs;  // [D][kLd]
  float* ys;  // [O][kLd] (backward)
  float* w1;  // [D][kLdW]
  float* wd;  // [O][kLdD]
  float* hs;  // one to three [kHid][kLd]

  // `tiles` buffers of rows and `weights` of weights; the first of each is in
  // use.
  __device__ Tile(const FfnParams& f, float* sm, bool bwd, int tiles, int weights) : p(f) {
    xs = sm;
    ys = xs + f.d * kLd;
    w1 = sm + tiles * (f.d + (bwd ? f.o : 0)) * kLd;
    wd = w1 + f.d * kLdW;
    hs = w1 + weights * weight_floats();
  }
  __device__ int weight_floats() const { return p.d * kLdW + p.o * kLdD; }

  // Rows from r0 on, transposed; zeros past the last. A warp's copies go to
  // 8 columns x 4 rows: 32 banks.
  __device__ void stage_rows(float* dst, const float* src, int64_t stride, int cols, int64_t r0) {
    const int lane = threadIdx.x & 31;
    for (int r = (threadIdx.x >> 5) * 4 + (lane >> 3); r < kRows; r += kThreads / 8) {
      const bool on = r0 + r < p.n;
      const float* from = on ? src + (r0 + r) * stride : src;
      for (int c = lane & 7; c < cols; c += 8) copy4(dst + c * kLd + r, from + c, on);
    }
  }

  // A chunk's weights, zeros past the last hidden value.
  __device__ void stage_weights(float* to1, float* tod, int h0) {
    const int lane = threadIdx.x & 31;
    {
      const int r = (threadIdx.x >> 5) * 4 + (lane >> 3);
      const bool on = h0 + r < p.h;
      const int64_t from = on ? static_cast<int64_t>(h0 + r) * p.d : 0;
      const float* wg = static_cast<const float*>(p.wg) + from;
      const float* wu = static_cast<const float*>(p.wu) + from;
      float* to = to1 + (r >> 1) * 4 + (r & 1);
      for (int c = lane & 7; c < p.d; c += 8) {
        copy4(to + c * kLdW, wg + c, on);
        copy4(to + c * kLdW + 2, wu + c, on);
      }
    }
    const bool on = h0 + lane < p.h;
    const float* w = static_cast<const float*>(p.wd) + (on ? h0 + lane : 0);
    for (int r = threadIdx.x >> 5; r < p.o; r += kThreads / 32)
      copy4(tod + r * kLdD + lane, w + static_cast<int64_t>(r) * p.h, on);
  }

  __device__ static void load_rows(const float* src, F2 (&v)[kR / 2]) {
    if constexpr (kR == 2) {
      const float2 q = *reinterpret_cast<const float2*>(src);
      v[0] = F2(q.x, q.y);
    } else {
#pragma unroll
      for (int i = 0; i < kR / 4; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(src + 4 * i);
        v[2 * i] = F2(q.x, q.y), v[2 * i + 1] = F2(q.z, q.w);
      }
    }
  }

  // This thread's kR rows of two hidden values: H to hs (kH), dG and dU to the
  // next two (kBwd).
  template <bool kBwd, bool kH>
  __device__ void hidden() {
    const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
    F2 g[2][kR / 2], u[2][kR / 2], dh[2][kR / 2];
#pragma unroll
    for (int i = 0; i < kR / 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) g[j][i] = u[j][i] = dh[j][i] = F2(0.f, 0.f);
#pragma unroll 2
    for (int k = 0; k < p.d; ++k) {
      F2 x[kR / 2];
      load_rows(xs + k * kLd + tr * kR, x);
      const float4 w = *reinterpret_cast<const float4*>(w1 + k * kLdW + 4 * tc);
      const F2 w0(w.x, w.x), wb(w.y, w.y), w2(w.z, w.z), w3(w.w, w.w);
#pragma unroll
      for (int i = 0; i < kR / 2; ++i) {
        g[0][i] = fma2(x[i], w0, g[0][i]);
        g[1][i] = fma2(x[i], wb, g[1][i]);
        u[0][i] = fma2(x[i], w2, u[0][i]);
        u[1][i] = fma2(x[i], w3, u[1][i]);
      }
    }
    if constexpr (kBwd) {
#pragma unroll 2
      for (int k = 0; k < p.o; ++k) {
        F2 y[kR / 2];
        load_rows(ys + k * kLd + tr * kR, y);
        const float2 w = *reinterpret_cast<const float2*>(wd + k * kLdD + 2 * tc);
        const F2 w0(w.x, w.x), wb(w.y, w.y);
#pragma unroll
        for (int i = 0; i < kR / 2; ++i) {
          dh[0][i] = fma2(y[i], w0, dh[0][i]);
          dh[1][i] = fma2(y[i], wb, dh[1][i]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* to = hs + (2 * tc + j) * kLd + tr * kR;
#pragma unroll
      for (int i = 0; i < kR / 2; ++i) {
        float ga, gb, ua, ub, da, db;
        g[j][i].get(ga, gb);
        u[j][i].get(ua, ub);
        const float sa = sigmoid(ga), sb = sigmoid(gb), aa = ga * sa, ab = gb * sb;
        if constexpr (kH) *reinterpret_cast<float2*>(to + 2 * i) = make_float2(aa * ua, ab * ub);
        if constexpr (kBwd) {
          dh[j][i].get(da, db);
          float* next = to + (kH ? kHid * kLd : 0);
          *reinterpret_cast<float2*>(next + 2 * i) =
              make_float2((sa + aa * (1.f - sa)) * ua * da, (sb + ab * (1.f - sb)) * ub * db);
          *reinterpret_cast<float2*>(next + kHid * kLd + 2 * i) = make_float2(da * aa, db * ab);
        }
      }
    }
  }

  __device__ static float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }
};

// Y (forward) or dX (backward): one tile of rows per block, all of H; thread
// column tc has output columns tc + 16 j.
template <int kR, bool kBwd, int kCols>
__global__ void __launch_bounds__(kThreads) ffn_rows_kernel(const FfnParams p, int buffers) {
  extern __shared__ __align__(16) float sm[];
  Tile<kR> t(p, sm, kBwd, 1, buffers);
  constexpr int kLd = t.kLd;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * t.kRows;
  t.stage_rows(t.xs, static_cast<const float*>(p.x), p.x_stride, p.d, r0);
  if constexpr (kBwd) t.stage_rows(t.ys, static_cast<const float*>(p.dy), p.dy_stride, p.o, r0);
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
  const int out = kBwd ? p.d : p.o;
  F2 acc[kCols][kR / 2];
#pragma unroll
  for (int j = 0; j < kCols; ++j)
#pragma unroll
    for (int i = 0; i < kR / 2; ++i) acc[j][i] = F2(0.f, 0.f);
  // With two buffers, the next chunk's weights are on their way under this
  // one's products.
  const int size = t.weight_floats();
  float* next = t.w1 + (buffers - 1) * size;
  t.stage_weights(t.w1, t.wd, 0);
  copies_commit();
  for (int h0 = 0; h0 < p.h; h0 += kHid) {
    if (buffers == 2 && h0 + kHid < p.h) t.stage_weights(next, next + p.d * kLdW, h0 + kHid);
    copies_commit();
    copies_wait<1>();
    __syncthreads();
    t.template hidden<kBwd, !kBwd>();
    __syncthreads();
    for (int k = 0; k < kHid; k += 2) {
      constexpr int kPairs = kBwd ? 4 : 2;  // H of both, or dG of both and dU of both
      F2 h[kPairs][kR / 2];
#pragma unroll
      for (int q = 0; q < kPairs; ++q)
        t.load_rows(t.hs + ((q >> 1) * kHid + k + (q & 1)) * kLd + tr * kR, h[q]);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int c = tc + 16 * j;
        if (c < out) {
          if constexpr (kBwd) {
            const float4 w = *reinterpret_cast<const float4*>(t.w1 + c * kLdW + 2 * k);
            const F2 w0(w.x, w.x), wb(w.y, w.y), w2(w.z, w.z), w3(w.w, w.w);
#pragma unroll
            for (int i = 0; i < kR / 2; ++i)
              acc[j][i] = fma2(h[3][i], w3, fma2(h[2][i], w2, fma2(h[1][i], wb, fma2(h[0][i], w0, acc[j][i]))));
          } else {
            const float2 w = *reinterpret_cast<const float2*>(t.wd + c * kLdD + k);
            const F2 w0(w.x, w.x), wb(w.y, w.y);
#pragma unroll
            for (int i = 0; i < kR / 2; ++i)
              acc[j][i] = fma2(h[1][i], wb, fma2(h[0][i], w0, acc[j][i]));
          }
        }
      }
    }
    __syncthreads();
    if (buffers == 2) {
      float* const w = t.w1;
      t.w1 = next, t.wd = next + p.d * kLdW, next = w;
    } else if (h0 + kHid < p.h) {
      t.stage_weights(t.w1, t.wd, h0 + kHid);
      copies_commit();
    }
  }
  float* y = static_cast<float*>(p.y);
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    const int c = tc + 16 * j;
#pragma unroll
    for (int i = 0; i < kR / 2; ++i) {
      float a, b;
      acc[j][i].get(a, b);
      const int64_t r = r0 + tr * kR + 2 * i;
      if (c < out && r < p.n) y[r * out + c] = a;
      if (c < out && r + 1 < p.n) y[(r + 1) * out + c] = b;
    }
  }
}

// Weights' gradients of one chunk of H (blockIdx.x) over one slice of the
// rows (blockIdx.y): scratch[slice][dWg [H, D] | dWu [H, D] | dWd^T [H, O]].
// Thread -> hidden values 2 th, 2 th + 1 and columns tc + 16 j; rows go in
// pairs, even and odd ones summed apart until the end.
template <int kR, int kCols>
__global__ void __launch_bounds__(kThreads) ffn_weights_kernel(const FfnParams p, int buffers) {
  extern __shared__ __align__(16) float sm[];
  Tile<kR> t(p, sm, true, buffers, 1);
  constexpr int kLd = t.kLd;
  const int h0 = blockIdx.x * kHid;
  auto stage = [&](float* to, int64_t r0) {
    t.stage_rows(to, static_cast<const float*>(p.x), p.x_stride, p.d, r0);
    t.stage_rows(to + p.d * kLd, static_cast<const float*>(p.dy), p.dy_stride, p.o, r0);
    copies_commit();
  };
  t.stage_weights(t.w1, t.wd, h0);
  // With two buffers, the next rows are on their way under this tile's products.
  float* next = t.xs + (buffers - 1) * (p.d + p.o) * kLd;
  const int64_t step = static_cast<int64_t>(gridDim.y) * t.kRows;
  stage(t.xs, static_cast<int64_t>(blockIdx.y) * t.kRows);
  const int th = threadIdx.x >> 4, tc = threadIdx.x & 15;
  F2 ag[2][kCols], au[2][kCols], ad[2][kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j)
#pragma unroll
    for (int q = 0; q < 2; ++q) ag[q][j] = au[q][j] = ad[q][j] = F2(0.f, 0.f);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * t.kRows; r0 < p.n; r0 += step) {
    if (buffers == 2 && r0 + step < p.n) {
      stage(next, r0 + step);
    } else {
      copies_commit();
    }
    copies_wait<1>();
    __syncthreads();
    t.template hidden<true, true>();
    __syncthreads();
#pragma unroll 2
    for (int r = 0; r < t.kRows; r += 4) {
      F2 v[6][2];  // H, dG, dU of both hidden values
#pragma unroll
      for (int q = 0; q < 6; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(
            t.hs + ((q >> 1) * kHid + 2 * th + (q & 1)) * kLd + r);
        v[q][0] = F2(f.x, f.y), v[q][1] = F2(f.z, f.w);
      }
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int c = tc + 16 * j;
        if (c < p.d) {
          const float4 f = *reinterpret_cast<const float4*>(t.xs + c * kLd + r);
          const F2 a(f.x, f.y), b(f.z, f.w);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            ag[q][j] = fma2(v[2 + q][1], b, fma2(v[2 + q][0], a, ag[q][j]));
            au[q][j] = fma2(v[4 + q][1], b, fma2(v[4 + q][0], a, au[q][j]));
          }
        }
        if (c < p.o) {
          const float4 f = *reinterpret_cast<const float4*>(t.ys + c * kLd + r);
          const F2 a(f.x, f.y), b(f.z, f.w);
#pragma unroll
          for (int q = 0; q < 2; ++q) ad[q][j] = fma2(v[q][1], b, fma2(v[q][0], a, ad[q][j]));
        }
      }
    }
    __syncthreads();
    if (buffers == 2) {
      float* const x = t.xs;
      t.xs = next, t.ys = next + p.d * kLd, next = x;
    } else if (r0 + step < p.n) {
      stage(t.xs, r0 + step);
    }
  }
  const int64_t hd = static_cast<int64_t>(p.h) * p.d;
  float* out = p.scratch + blockIdx.y * (2 * hd + static_cast<int64_t>(p.h) * p.o);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int64_t hid = h0 + 2 * th + q;
    if (hid >= p.h) continue;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int c = tc + 16 * j;
      float a, b;
      if (c < p.d) {
        ag[q][j].get(a, b);
        out[hid * p.d + c] = a + b;
        au[q][j].get(a, b);
        out[hd + hid * p.d + c] = a + b;
      }
      if (c < p.o) {
        ad[q][j].get(a, b);
        out[2 * hd + hid * p.o + c] = a + b;
      }
    }
  }
}

// Sums the slices in a fixed order and writes the gradients in the weights'
// layouts: 32 values a block, the slices dealt to its eight warps.
__global__ void __launch_bounds__(kThreads) ffn_weights_sum_kernel(const FfnParams p, int slices) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t hd = static_cast<int64_t>(p.h) * p.d, all = 2 * hd + static_cast<int64_t>(p.h) * p.o;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (e < all) {
#pragma unroll 4
    for (int s = warp; s < slices; s += 8) sum += p.scratch[s * all + e];
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp > 0 || e >= all) return;
  for (int w = 1; w < 8; ++w) sum += part[w][lane];
  if (e < hd) {
    static_cast<float*>(p.dwg)[e] = sum;
  } else if (e < 2 * hd) {
    static_cast<float*>(p.dwu)[e - hd] = sum;
  } else {
    const int64_t i = (e - 2 * hd) / p.o, j = (e - 2 * hd) - i * p.o;
    static_cast<float*>(p.dwd)[j * p.h + i] = sum;
  }
}

// Rows per thread: as many as shared memory holds, the wider of D and O
// deciding (its columns are then at most 4, 8 and 16 to a thread too).
int rows_per_thread(int d, int o) {
  const int w = std::max(d, o);
  return w <= 64 ? 8 : w <= 128 ? 4 : 2;
}

int tile_smem(const FfnParams& p, int r, bool bwd, int hidden, int tiles, int weights) {
  return 4 * ((tiles * (p.d + (bwd ? p.o : 0)) + hidden * kHid) * rows_ld(r) +
              weights * (p.d * kLdW + p.o * kLdD));
}
// All that a block can have; the kernels' limit at every size, since it belongs
// to the kernel and another thread may be launching it at another size.
constexpr int kMostSmem = 227 * 1024;

int ffn_slices(int64_t n, int d, int h, int o) {
  const int64_t chunks = ceil_div(h, kHid), tiles = ceil_div<int64_t>(n, 16 * rows_per_thread(d, o));
  return static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(tiles, ceil_div<int64_t>(2 * sm_count(), chunks))));
}

int64_t weights_floats(int64_t n, int d, int h, int o) {
  return ffn_slices(n, d, h, o) * static_cast<int64_t>(h) * (2 * d + o);
}

template <int kR, bool kBwd, int kCols>
int launch_rows(const FfnParams& p, cudaStream_t s) {
  int smem = tile_smem(p, kR, kBwd, kBwd ? 2 : 1, 1, 2), buffers = 2;
  if (p.h <= kHid || smem > kMostSmem) smem = tile_smem(p, kR, kBwd, kBwd ? 2 : 1, 1, 1), buffers = 1;
  TGS_CUDA(cudaFuncSetAttribute(ffn_rows_kernel<kR, kBwd, kCols>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
  ffn_rows_kernel<kR, kBwd, kCols>
      <<<static_cast<unsigned>(ceil_div<int64_t>(p.n, 16 * kR)), kThreads, smem, s>>>(p, buffers);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

template <bool kBwd>
int rows_f32(const FfnParams& p, cudaStream_t s) {
  const int out = kBwd ? p.d : p.o;
  switch (rows_per_thread(p.d, p.o)) {
    case 8: return out <= 16 ? launch_rows<8, kBwd, 1>(p, s) : launch_rows<8, kBwd, 4>(p, s);
    case 4: return out <= 32 ? launch_rows<4, kBwd, 2>(p, s) : launch_rows<4, kBwd, 8>(p, s);
    default: return out <= 64 ? launch_rows<2, kBwd, 4>(p, s) : launch_rows<2, kBwd, 16>(p, s);
  }
}

template <int kR, int kCols>
int launch_weights(const FfnParams& p, int slices, cudaStream_t s) {
  int smem = tile_smem(p, kR, true, 3, 2, 1), buffers = 2;
  if (smem > kMostSmem) smem = tile_smem(p, kR, true, 3, 1, 1), buffers = 1;
  TGS_CUDA(cudaFuncSetAttribute(ffn_weights_kernel<kR, kCols>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
  ffn_weights_kernel<kR, kCols><<<dim3(ceil_div(p.h, kHid), slices), kThreads, smem, s>>>(p, buffers);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

// Whether a 32-bit call takes the tensor cores: by the multiply-adds of a row.
// Their fixed work on each matrix (splitting, a trip through L2) pays for
// itself from about 12,000 on, at any number of rows. 100,000 rows, forward and
// forward + backward, fp32 pipes against tensor cores: 35 -> 96 -> 3 (7,008) 63
// and 397 us against 119 and 507; 48 -> 96 -> 48 (13,824) 99 and 617 against
// 129 and 493; 128 -> 256 -> 128 (98,304) 807 and 4127 against 300 and 1207.
bool wide_f32(int d, int h, int o) {
  return static_cast<int64_t>(h) * (2 * d + o) >= 12288;
}

int sum_slices(const FfnParams& p, int slices, cudaStream_t s) {
  const int64_t all = static_cast<int64_t>(p.h) * (2 * p.d + p.o);
  ffn_weights_sum_kernel<<<static_cast<unsigned>(ceil_div<int64_t>(all, 32)), kThreads, 0, s>>>(p, slices);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

int ffn_backward_f32(const FfnParams& p, cudaStream_t s) {
  if (wide_f32(p.d, p.h, p.o)) {
    if (int rc = ffn_tc32_run(p, true, s)) return rc;
    return p.dwg ? sum_slices(p, tc32_slices(p.n, p.d, p.h, p.o), s) : TGS_OK;
  }
  if (p.y) {
    if (int rc = rows_f32<true>(p, s)) return rc;
  }
  if (!p.dwg) return TGS_OK;
  const int slices = ffn_slices(p.n, p.d, p.h, p.o);
  int rc = TGS_OK;
  switch (rows_per_thread(p.d, p.o)) {
    case 8: rc = launch_weights<8, 4>(p, slices, s); break;
    case 4: rc = launch_weights<4, 8>(p, slices, s); break;
    default: rc = launch_weights<2, 16>(p, slices, s); break;
  }
  return rc ? rc : sum_slices(p, slices, s);
}

bool aligned_rows(const TgsFfnArgs& a, const void* p, int64_t stride) {
  return a.n == 0 || a.dtype == TGS_F32 || (stride > 0 && stride % 8 == 0 && aligned16(p));
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
  if (wide_f32(d, h, o)) return tc32_scratch_floats(n, d, h, o, backward != 0);
  return backward ? weights_floats(n, d, h, o) : 0;
}

extern "C" int tgs_ffn_fwd(const TgsFfnArgs* a, void* stream) {
  launches() = 0;
  if (int rc = check_ffn(a, "tgs_ffn_fwd")) return rc;
  if (a->n == 0) return TGS_OK;
  TGS_CHECK_ARG(a->y != nullptr, "tgs_ffn_fwd: NULL pointer");
  TGS_CHECK_ARG(aligned_rows(*a, a->x, a->x_stride) && aligned16(a->y) && aligned16(a->scratch),
                "tgs_ffn_fwd: y, scratch or the rows of x are not 16-byte aligned (stride %lld)",
                static_cast<long long>(a->x_stride));
  TGS_CHECK_ARG(a->scratch || !tgs_ffn_scratch_floats(a->n, a->d, a->h, a->o, a->dtype, 0),
                "tgs_ffn_fwd: scratch is NULL");
  const FfnParams p = ffn_params(*a);
  cudaStream_t s = as_stream(stream);
  if (a->dtype == TGS_BF16) return ffn_tc_forward(p, s);
  return wide_f32(p.d, p.h, p.o) ? ffn_tc32_run(p, false, s) : rows_f32<false>(p, s);
}

extern "C" int tgs_ffn_bwd(const TgsFfnBwdArgs* b, void* stream) {
  launches() = 0;
  TGS_CHECK_ARG(b != nullptr, "tgs_ffn_bwd: args is NULL");
  const TgsFfnArgs& a = b->fwd;
  if (int rc = check_ffn(&a, "tgs_ffn_bwd")) return rc;
  const bool weights = b->v_w_gate || b->v_w_up || b->v_w_down;
  TGS_CHECK_ARG(!weights || (b->v_w_gate && b->v_w_up && b->v_w_down),
                "tgs_ffn_bwd: the weights' gradients are all given or none");
  TGS_CHECK_ARG(a.n == 0 || (b->v_y && (b->v_x || weights)), "tgs_ffn_bwd: NULL pointer");
  TGS_CHECK_ARG(a.n <= 1 || b->v_y_stride >= a.o, "tgs_ffn_bwd: rows of v_y overlap");
  TGS_CHECK_ARG(aligned_rows(a, a.x, a.x_stride) && aligned_rows(a, b->v_y, b->v_y_stride) &&
                    aligned16(b->v_x) && aligned16(a.scratch),
                "tgs_ffn_bwd: v_x, scratch or the rows of x or v_y are not 16-byte aligned (strides %lld, %lld)",
                static_cast<long long>(a.x_stride), static_cast<long long>(b->v_y_stride));
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
