// Gated feed-forward block in 32 bits on the tensor cores, for large calls; the
// formulas stand in tgs_ffn.cu.
//
// A 32-bit number is the sum of three bf16 numbers up to 2^-24 of it (8 bits
// each, every difference exact), so a 32-bit product is six bf16 products,
// those of parts that weigh 2^-16 or more. Tiles are split on their way into
// shared memory: one stage holds both operands' three parts, 96 KB. That
// leaves no room for a whole row's widths and hidden values, so here they do
// go through memory, in batches of rows small enough to stay in L2: one launch
// makes the hidden values, one the output, one the weights' gradients.
//
// A block makes one 128 x 128 tile of a product. Sixteen warps load and split,
// and store the result; one issues the matrix instructions. The accumulators
// round towards zero: 96 additions to one left 2.4e-6 of the result, 192
// 5.7e-6. So a stage's products, the smallest first, get accumulators of their
// own (two take turns) and are added in registers, where additions round to
// the nearest.
#include "tgs_ffn.cuh"
#include "tgs_tc.cuh"

namespace tgs {
namespace {

constexpr int kWorkers = 512;
constexpr int kThreads32 = kWorkers + 32;
constexpr int kTile = 128;
constexpr int kStep = 64;             // contracted values per stage
constexpr int kPart = kBlockBytes;    // one operand's part of a stage
constexpr int kStage = 6 * kPart;     // A's three parts, then B's
constexpr int kUnits = 1024 / kWorkers;  // of eight values, per operand, thread and stage

enum : int { kHidden = 0, kHiddenBwd = 1, kOutput = 2, kWeights = 3 };

// A row-major matrix of which tiles are taken.
struct Mat {
  const float* p;
  int64_t ld;
  int64_t rows;
  int cols;
};

// One contraction. Operands with `mn` have the contracted index along their
// rows, the others along their columns.
struct Term {
  Mat a, b, b2;  // b2: rows 64-127 of b's tile (kHidden)
  int k;         // contracted length
};

struct Tc32Params {
  Term t[3];
  int terms;
  float* out[3];     // hidden: h, dG, dU; output: one; weights: the slices
  int64_t out_ld;
  int64_t rows;      // of this batch
  int64_t per_slice; // rows of a slice (weights), a multiple of kStep
  int h, d, o;
  int stages, first; // first: the slices are written, not added to
  int32_t* err;
};

// Eight values of a row.
struct Unit {
  float v[8];
};

__device__ __forceinline__ Unit load_values(const Mat& m, int64_t row, int64_t row_end, int col,
                                            bool vec) {
  Unit u;
  const float* p = m.p + row * m.ld + col;
  if (row < row_end && col + 8 <= m.cols && vec) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    u.v[0] = a.x, u.v[1] = a.y, u.v[2] = a.z, u.v[3] = a.w;
    u.v[4] = b.x, u.v[5] = b.y, u.v[6] = b.z, u.v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) u.v[i] = row < row_end && col + i < m.cols ? p[i] : 0.f;
  }
  return u;
}

// The three parts to their places.
__device__ __forceinline__ void store_parts(uint32_t at, const Unit& u) {
  uint32_t q[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = u.v[2 * i], b = u.v[2 * i + 1];
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      const uint32_t r = pack_bf16(a, b);
      q[part][i] = r;
      a -= __uint_as_float(r << 16), b -= __uint_as_float(r & 0xffff0000u);
    }
  }
#pragma unroll
  for (int part = 0; part < 3; ++part)
    st_shared16(at + part * kPart, make_uint4(q[part][0], q[part][1], q[part][2], q[part][3]));
}

__device__ __forceinline__ bool vec_rows(const Mat& m) { return aligned16(m.p) && m.ld % 4 == 0; }

template <int kJob>
__global__ void __launch_bounds__(kThreads32) ffn_tc32_kernel(const __grid_constant__ Tc32Params p) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[2], done[2], drained[2];
  __shared__ uint32_t tmem_slot;
  constexpr bool kMn = kJob == kWeights;           // both operands by rows
  constexpr bool kHid = kJob <= kHiddenBwd;
  constexpr uint32_t kCols = 256;  // two accumulators
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  // This block's tile: rows m0 of A's side, columns n0 of B's.
  int64_t m0 = 0, k_begin = 0, k_end = 0;  // k_begin, k_end: rows of the slice (weights)
  int n0 = 0, n = kTile, which = 0;
  if constexpr (kHid) {
    m0 = static_cast<int64_t>(blockIdx.x) * kTile, n0 = blockIdx.y * 64;
  } else if constexpr (kJob == kOutput) {
    m0 = static_cast<int64_t>(blockIdx.x) * kTile, n0 = blockIdx.y * kTile;
    n = min(kTile, (static_cast<int>(p.out_ld) - n0 + 15) & ~15);
  } else {
    const int hid_tiles = (p.h + kTile - 1) / kTile, d_tiles = (p.d + kTile - 1) / kTile;
    const int o_tiles = (p.o + kTile - 1) / kTile;
    int y = blockIdx.y;
    const int each = hid_tiles * d_tiles;
    which = min(y / each, 2), y -= which * each;
    const int tiles = which < 2 ? d_tiles : o_tiles, width = which < 2 ? p.d : p.o;
    m0 = (y / tiles) * kTile, n0 = (y % tiles) * kTile;
    n = min(kTile, (width - n0 + 15) & ~15);
    k_begin = static_cast<int64_t>(blockIdx.x) * p.per_slice;
    k_end = min64(p.rows, k_begin + p.per_slice);
  }
  // Stages of this block, over its terms.
  int total = 0;
  if constexpr (kMn) {
    total = k_end > k_begin ? static_cast<int>((k_end - k_begin + kStep - 1) / kStep) : 0;
  } else {
    for (int t = 0; t < p.terms; ++t) total += (p.t[t].k + kStep - 1) / kStep;
  }

  if (warp == kWorkers / 32) {
    tmem_alloc(&tmem_slot, kCols);
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&full[i], kWorkers / 32), mbar_init(&done[i], 1);
        mbar_init(&drained[i], kWorkers / 32);
      }
      fence_mbar_init();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t acc = tmem_slot;
  bool ok = true;
  auto wait = [&](uint64_t* bar, int phase) {
    if (ok && !tc_wait(bar, phase & 1)) {
      ok = false;
      report_error(p.err, TGS_DEV_WAIT_TIMEOUT, blockIdx.x, threadIdx.x);
    }
  };

  if (warp < kWorkers / 32) {
    const int tid = threadIdx.x;
    const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;
    const int row = (warp & 3) * 32 + lane, part = warp >> 2;  // a quarter of the columns
    // hidden: 16 columns of G, U and dH; else 32 of the tile
    float sum[3][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[0][i] = sum[1][i] = sum[2][i] = 0.f;
    auto add = [&](int col, float (&to)[16]) {
      float v[16];
      tmem_ld(acc + quarter + col, v);
      tmem_wait_ld(v);
#pragma unroll
      for (int i = 0; i < 16; ++i) to[i] += v[i];
    };
    // Adds stage s, which belongs to term `of`.
    auto drain = [&](int s, int of) {
      wait(&done[s & 1], s >> 1);
      tc_fence_after();
      const int at = (s & 1) * 128;
      if constexpr (kHid) {
        if (kJob == kHiddenBwd && of == 1) {
          add(at + 16 * part, sum[2]);
        } else {
          add(at + 16 * part, sum[0]);
          add(at + 64 + 16 * part, sum[1]);
        }
      } else {
        if (32 * part < n) add(at + 32 * part, sum[0]);
        if (32 * part + 16 < n) add(at + 32 * part + 16, sum[1]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[s & 1]);
    };
    int term = which, k0 = 0;
    Unit a[kUnits], b[kUnits];
    auto load = [&] {
      const Term& t = p.t[term];
      if constexpr (kMn) {  // [64 rows][128 columns] of each
        const int64_t r0 = k_begin + k0;
        const bool va = vec_rows(t.a), vb = vec_rows(t.b);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int e = tid + i * kWorkers, r = e >> 4, unit = e & 15;
          a[i] = load_values(t.a, r0 + r, k_end, static_cast<int>(m0) + unit * 8, va);
          b[i] = load_values(t.b, r0 + r, k_end, n0 + unit * 8, vb);
        }
      } else {
        const bool va = vec_rows(t.a), vb = vec_rows(t.b) && (!kHid || vec_rows(t.b2));
        // B by rows: the second term of the hidden values, and dX's terms
        const bool b_mn = kJob == kHiddenBwd ? term == 1 : kJob == kOutput && p.d > 0;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          const int e = tid + i * kWorkers;
          a[i] = load_values(t.a, m0 + (e >> 3), t.a.rows, k0 + (e & 7) * 8, va);
          if (b_mn) {
            b[i] = load_values(t.b, k0 + (e >> 4), t.b.rows, n0 + (e & 15) * 8, vb);
          } else if (kHid && (e >> 3) >= 64) {
            b[i] = load_values(t.b2, n0 + (e >> 3) - 64, t.b2.rows, k0 + (e & 7) * 8, vb);
          } else {
            const int64_t end = kHid ? t.b.rows : min64(t.b.rows, n0 + n);
            b[i] = load_values(t.b, n0 + (e >> 3), end, k0 + (e & 7) * 8, vb);
          }
        }
      }
      k0 += kStep;
      if (!kMn && k0 >= t.k) k0 = 0, ++term;
    };
    int used = term, before = term;
    if (total > 0) load();
    for (int s = 0; s < total; ++s) {
      // the stage that last used this half of shared memory has been drained
      const uint32_t to = base + (p.stages == 2 ? s & 1 : 0) * kStage;
      const bool b_mn = kMn || (kJob == kHiddenBwd ? used == 1 : kJob == kOutput && p.d > 0);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int e = tid + i * kWorkers;
        const uint32_t k_at = unit_offset(e >> 3, e & 7);
        const uint32_t mn_at = ((e >> 3) & 1) * (kPart / 2) + unit_offset(e >> 4, e & 7);
        store_parts(to + (kMn ? mn_at : k_at), a[i]);
        store_parts(to + 3 * kPart + (b_mn ? mn_at : k_at), b[i]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s & 1]);
      const int of = used;
      used = term;
      if (s + 1 < total) load();
      if (s > 0) drain(s - 1, before);
      before = of;
    }
    if (total > 0) drain(total - 1, before);
    const int64_t r = m0 + row;
    if constexpr (kMn) {
      if (r < p.h) {
        const int64_t hd = static_cast<int64_t>(p.h) * p.d;
        const int width = which < 2 ? p.d : p.o;
        float* to = p.out[0] + blockIdx.x * (2 * hd + static_cast<int64_t>(p.h) * p.o) + which * hd +
                    r * width;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int c = n0 + 32 * part + i;
          const float v = sum[i >> 4][i & 15];
          if (c < width) to[c] = p.first ? v : to[c] + v;
        }
      }
    } else if constexpr (kHid) {
      const int c = n0 + 16 * part;
      if (r < p.rows && c < p.h) {
        float* to = p.out[0] + r * p.out_ld + c;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          float h[4], dg[4], du[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = sum[0][i + k], u = sum[1][i + k], d = sum[2][i + k];
            const float sg = __fdividef(1.f, 1.f + __expf(-x)), act = x * sg;
            h[k] = act * u;
            dg[k] = d * u * (sg + act * (1.f - sg));
            du[k] = d * act;
          }
          *reinterpret_cast<float4*>(to + i) = make_float4(h[0], h[1], h[2], h[3]);
          if constexpr (kJob == kHiddenBwd) {
            *reinterpret_cast<float4*>(p.out[1] + (to - p.out[0]) + i) =
                make_float4(dg[0], dg[1], dg[2], dg[3]);
            *reinterpret_cast<float4*>(p.out[2] + (to - p.out[0]) + i) =
                make_float4(du[0], du[1], du[2], du[3]);
          }
        }
      }
    } else {
      const int width = static_cast<int>(p.out_ld), c = n0 + 32 * part;
      if (r < p.rows) {
        float* to = p.out[0] + r * p.out_ld + c;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (c + i < width) to[i] = sum[i >> 4][i & 15];
      }
    }
  } else {
    // Parts of A and B, the smallest products first.
    constexpr int kPa[6] = {0, 1, 2, 0, 1, 0}, kPb[6] = {2, 1, 0, 1, 0, 0};
    int term = which, k0 = 0;
    for (int s = 0; s < total; ++s) {
      const int st = s & 1;
      if (s >= 2) wait(&drained[st], (s >> 1) - 1);
      wait(&full[st], s >> 1);
      tc_fence_after();
      const uint32_t from = base + (p.stages == 2 ? st : 0) * kStage;
      const bool b_mn = kMn || (kJob == kHiddenBwd ? term == 1 : kJob == kOutput && p.d > 0);
      const int k = kMn ? kStep : p.t[term].k;
      const int steps = kMn ? 4 : min(4, (k - k0 + 15) >> 4);
      const uint32_t to = acc + st * 128;
      const uint32_t id = tc_idesc(kJob == kHiddenBwd && term == 1 ? 64 : n, kMn, b_mn);
      const uint32_t da = kMn ? desc_mn(from, kPart / 2) : desc_k(from);
      const uint32_t db = b_mn ? desc_mn(from + 3 * kPart, kPart / 2) : desc_k(from + 3 * kPart);
      const uint32_t sa = kMn ? kStepMn : kStepK, sb = b_mn ? kStepMn : kStepK;
#pragma unroll
      for (int q = 0; q < 6; ++q)
        tc_mma_steps<4>(to, da + kPa[q] * (kPart >> 4), sa, db + kPb[q] * (kPart >> 4), sb, id, steps,
                        q > 0);
      tc_commit(&done[st]);
      if (!kMn && (k0 += kStep) >= k) k0 = 0, ++term;
    }
    if (total > 0) wait(&done[(total - 1) & 1], (total - 1) >> 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kWorkers / 32) {
    tc_fence_after();
    tmem_free(acc, kCols);
  }
}

template <int kJob>
int launch32(Tc32Params p, dim3 grid, cudaStream_t s) {
  int total = kJob == kWeights ? 2 : 0;
  for (int t = 0; kJob != kWeights && t < p.terms; ++t) total += ceil_div(p.t[t].k, kStep);
  p.stages = total > 1 ? 2 : 1;
  const int smem = p.stages * kStage + 1024;
  TGS_CUDA(cudaFuncSetAttribute(ffn_tc32_kernel<kJob>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                smem));
  ffn_tc32_kernel<kJob><<<grid, kThreads32, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

// Rows of a batch: its three hidden matrices together take at most about 64 MB
// of the 126 MB of L2; batches of one size.
int64_t batch_rows(int64_t n, int h) {
  const int64_t tiles = ceil_div<int64_t>(n, kTile);
  const int64_t most = std::max<int64_t>(1, (16ll << 20) / (3 * ceil_div(h, 64) * 64) / kTile);
  return ceil_div(tiles, ceil_div(tiles, most)) * kTile;
}

int64_t padded(int h) { return ceil_div(h, 64) * 64; }

int weight_tiles(int d, int h, int o) {
  return ceil_div(h, kTile) * (2 * ceil_div(d, kTile) + ceil_div(o, kTile));
}

}  // namespace

int tc32_slices(int64_t n, int d, int h, int o) {
  const int64_t rows = std::min(n, batch_rows(n, h));
  const int64_t most = std::max(1, 2 * sm_count() / weight_tiles(d, h, o));
  return static_cast<int>(std::min<int64_t>(most, ceil_div<int64_t>(rows, 4 * kStep)));
}

// Floats of scratch: the hidden matrices of a batch, after `slices` partial
// gradients.
int64_t tc32_hidden_floats(int64_t n, int h, bool backward) {
  return batch_rows(n, h) * padded(h) * (backward ? 3 : 1);
}

int ffn_tc32_run(const FfnParams& f, bool backward, cudaStream_t s) {
  const int64_t hp = padded(f.h), batch = batch_rows(f.n, f.h);
  const int slices = tc32_slices(f.n, f.d, f.h, f.o);
  const int64_t partial = backward && f.dwg ? slices * static_cast<int64_t>(f.h) * (2 * f.d + f.o) : 0;
  float* hid = f.scratch + ceil_div<int64_t>(partial, 4) * 4;
  const float* wg = static_cast<const float*>(f.wg);
  const float* wu = static_cast<const float*>(f.wu);
  const float* wd = static_cast<const float*>(f.wd);
  const Mat mg{wg, f.d, f.h, f.d}, mu{wu, f.d, f.h, f.d}, md{wd, f.h, f.o, f.h};
  for (int64_t r0 = 0; r0 < f.n; r0 += batch) {
    const int64_t rows = std::min(batch, f.n - r0);
    const unsigned tiles = static_cast<unsigned>(ceil_div<int64_t>(rows, kTile));
    const Mat x{static_cast<const float*>(f.x) + r0 * f.x_stride, f.x_stride, rows, f.d};
    const Mat dy{static_cast<const float*>(f.dy) + (backward ? r0 * f.dy_stride : 0), f.dy_stride, rows,
                 f.o};
    Mat hm[3];  // h, dG, dU
    Tc32Params p{};
    p.rows = rows, p.h = f.h, p.err = f.err;
    p.out_ld = hp;
    for (int i = 0; i < 3; ++i) {
      p.out[i] = hid + i * batch * hp;
      hm[i] = Mat{p.out[i], hp, rows, f.h};
    }
    p.t[0] = Term{x, mg, mu, f.d};
    p.terms = 1;
    const dim3 grid(tiles, ceil_div(f.h, 64));
    if (!backward) {
      if (int rc = launch32<kHidden>(p, grid, s)) return rc;
    } else {
      p.t[1] = Term{dy, md, md, f.o};
      p.terms = 2;
      if (int rc = launch32<kHiddenBwd>(p, grid, s)) return rc;
    }
    Tc32Params q{};
    q.rows = rows, q.h = f.h, q.err = f.err;
    if (!backward || f.y) {
      const int out = backward ? f.d : f.o;
      q.out[0] = static_cast<float*>(f.y) + r0 * out;
      q.out_ld = out, q.d = backward;  // d > 0: B by rows
      if (backward) {
        q.t[0] = Term{hm[1], mg, mg, f.h};
        q.t[1] = Term{hm[2], mu, mu, f.h};
        q.terms = 2;
      } else {
        q.t[0] = Term{hm[0], md, md, f.h};
        q.terms = 1;
      }
      if (int rc = launch32<kOutput>(q, dim3(tiles, ceil_div(out, kTile)), s)) return rc;
    }
    if (partial) {
      q.t[0] = Term{hm[1], x, x, 0};
      q.t[1] = Term{hm[2], x, x, 0};
      q.t[2] = Term{hm[0], dy, dy, 0};
      q.terms = 3;
      q.d = f.d, q.o = f.o;
      q.out[0] = f.scratch;
      q.per_slice = ceil_div<int64_t>(ceil_div<int64_t>(rows, slices), kStep) * kStep;
      q.first = r0 == 0;
      if (int rc = launch32<kWeights>(q, dim3(slices, weight_tiles(f.d, f.h, f.o)), s)) return rc;
    }
  }
  return TGS_OK;
}

}  // namespace tgs
