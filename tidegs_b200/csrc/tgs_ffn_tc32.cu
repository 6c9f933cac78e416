// Gated feed-forward block in 32 bits on the tensor cores, for wide blocks; the
// formulas stand in tgs_ffn.cu.
//
// A 32-bit number is the sum of three bf16 numbers up to 2^-24 of it (8 bits
// each, every difference exact), so a 32-bit product is six bf16 products,
// those of parts that weigh 2^-16 or more. Three parts of whole rows, of the
// weights and of the hidden values do not fit beside one another in shared
// memory, so here each matrix is split once, into the operand blocks of
// tgs_tc.cuh, and goes through memory in batches of rows small enough to stay
// in L2: one launch splits the rows, one makes the hidden values (split again
// as they are stored), one the output, one the weights' gradients.
//
// A block makes one 128 x 128 tile of a product: one thread copies operand
// blocks (a stage is both operands' three parts, 96 KB), one warp issues the
// matrix instructions, eight add and store. The accumulators round towards
// zero: 96 additions to one left 2.4e-6 of the result, 192 5.7e-6. So a
// stage's products, the smallest first, get accumulators of their own (two
// take turns) and are added in registers, where additions round to the
// nearest. Bound: the matrix instructions, 24 to a stage, and what stands
// before a tile's first and after its last: 50,000 rows of 256 -> 512 -> 256
// forward 390 us (605 TFLOP/s of bf16 products), backward 1344 us. Parts of
// values below 2^-100 fall out of bf16's range, and the further parts of an
// infinity, or of a value that rounds to one in bf16 (from 3.396e38 on), are NaN.
#include "tgs_ffn.cuh"
#include "tgs_tc.cuh"

namespace tgs {
namespace {

constexpr int kAdders = 256;
constexpr int kThreads32 = kAdders + 64;
constexpr int kTile = 128;
constexpr int kStep = 64;             // contracted values per stage
constexpr int kPart = kBlockBytes;    // one operand's part of a stage
constexpr int kStage = 6 * kPart;     // A's three parts, then B's
constexpr int kBlock3 = 3 * kPart;    // a block's three parts, one after another

enum : int { kHidden = 0, kHiddenBwd = 1, kOutput = 2, kWeights = 3 };

// A matrix in split blocks of 128 rows x 64 columns: block (r, c) at index
// r x col_blocks + c. By its columns it is a K-major operand, by its rows (in
// halves of 64) an MN-major one.
struct Split {
  uint8_t* p;
  int col_blocks;
};

struct Tc32Params {
  Split x, dy, h, dg, du, gu, d;  // gu: block (j, c) has Wg's rows of chunk j, then Wu's
  float* out;        // the output's rows, or the slices of the gradients
  int64_t rows;      // of this batch
  int tiles;         // of 128 rows
  int per_slice;     // halves of tiles (64 rows) in a slice
  int width;         // of the output
  int hid, din, dout;  // H, D, O
  int bwd, first;    // first: the slices are written, not added to
  int32_t* err;
};

// The three parts of eight values to their places, `step` bytes apart.
template <class Store>
__device__ __forceinline__ void split8(const float (&v)[8], Store&& store) {
  uint32_t q[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      const uint32_t r = pack_bf16(a, b);
      q[part][i] = r;
      a -= __uint_as_float(r << 16), b -= __uint_as_float(r & 0xffff0000u);
    }
  }
#pragma unroll
  for (int part = 0; part < 3; ++part)
    store(part, make_uint4(q[part][0], q[part][1], q[part][2], q[part][3]));
}

// Splits a row-major matrix; block x of the grid is (row tile, column block).
// With `second`, rows 64-127 of a tile are the second matrix's (64 rows of each
// to a tile).
__global__ void __launch_bounds__(256) split_kernel(const float* first, const float* second,
                                                    int64_t ld, int64_t rows, int cols, Split to) {
  const int64_t tile = blockIdx.x / to.col_blocks;
  const int c = blockIdx.x % to.col_blocks;
  uint8_t* block = to.p + static_cast<int64_t>(blockIdx.x) * kBlock3;
  const bool vec = ld % 4 == 0 && aligned16(first) && (!second || aligned16(second));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x + 256 * i, r = e >> 3, unit = e & 7;
    const float* m = second && r >= 64 ? second : first;
    const int64_t row = second ? tile * 64 + (r & 63) : tile * kTile + r;
    const int col = c * kBlockCols + unit * 8;
    const float* p = m + row * ld + col;
    float v[8];
    if (row < rows && col + 8 <= cols && vec) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = row < rows && col + k < cols ? p[k] : 0.f;
    }
    split8(v, [&](int part, uint4 q) {
      *reinterpret_cast<uint4*>(block + part * kPart + unit_offset(r, unit)) = q;
    });
  }
}

// One stage of a tile's contraction: where its operands lie, in pieces of
// 64 rows (kHalf bytes each).
constexpr int kHalf = kPart / 2;
struct StagePlan {
  const uint8_t* a[2];  // first part of each piece
  const uint8_t* b[2];
  int a_pieces, b_pieces, steps;  // steps of 16
  bool b_mn;
  int n;
};

template <int kJob>
struct Tile32 {
  const Tc32Params& p;
  int m, n0, which, total, k_begin;

  __device__ __forceinline__ explicit Tile32(const Tc32Params& q) : p(q) {
    which = 0, k_begin = 0;
    if constexpr (kJob <= kHiddenBwd) {
      m = blockIdx.x, n0 = blockIdx.y;  // row tile, chunk
      total = p.x.col_blocks + (kJob == kHiddenBwd ? p.dy.col_blocks : 0);
    } else if constexpr (kJob == kOutput) {
      m = blockIdx.x, n0 = blockIdx.y;  // row tile, 128 columns
      total = p.bwd ? 2 * p.h.col_blocks : p.h.col_blocks;
    } else {
      const int hid_tiles = (p.hid + kTile - 1) / kTile, d_tiles = (p.din + kTile - 1) / kTile;
      const int each = hid_tiles * d_tiles;
      int y = blockIdx.y;
      which = min(y / each, 2), y -= which * each;  // dWg, dWu, dWd
      const int tiles = which < 2 ? d_tiles : (p.dout + kTile - 1) / kTile;
      m = y / tiles, n0 = y % tiles;  // 128 hidden values, 128 columns
      k_begin = blockIdx.x * p.per_slice;
      total = max(0, min(2 * p.tiles, k_begin + p.per_slice) - k_begin);
    }
  }

  // Columns of B's side.
  __device__ __forceinline__ int columns() const {
    if constexpr (kJob <= kHiddenBwd) return kTile;
    const int width = kJob == kOutput ? p.width : which < 2 ? p.din : p.dout;
    return min(kTile, (width - n0 * kTile + 15) & ~15);
  }

  __device__ __forceinline__ StagePlan stage(int s) const {
    auto block = [](const Split& t, int r, int c) {
      return t.p + (static_cast<int64_t>(r) * t.col_blocks + c) * kBlock3;
    };
    StagePlan q;
    q.n = columns();
    if constexpr (kJob == kWeights) {
      const Split& a = which == 0 ? p.dg : which == 1 ? p.du : p.h;
      const Split& b = which < 2 ? p.x : p.dy;
      const int half = k_begin + s, off = (half & 1) * kHalf;
      q.a[0] = block(a, half >> 1, 2 * m) + off;
      q.b[0] = block(b, half >> 1, 2 * n0) + off;
      q.a_pieces = 2 * m + 1 < a.col_blocks ? 2 : 1;
      q.b_pieces = q.n > 64 ? 2 : 1;
      q.a[1] = q.a[0] + kBlock3, q.b[1] = q.b[0] + kBlock3;
      q.b_mn = true, q.steps = 4;
    } else {
      const bool second = kJob == kHiddenBwd && s >= p.x.col_blocks;
      const int c = second ? s - p.x.col_blocks : s;
      int k;
      if constexpr (kJob == kOutput) {
        const int j = p.bwd ? s >> 1 : s;
        const Split& a = !p.bwd ? p.h : s & 1 ? p.du : p.dg;
        q.a[0] = block(a, m, j);
        k = p.hid - j * kStep;
        if (p.bwd) {  // Wg's or Wu's rows of the chunk, 64 columns a piece
          q.b[0] = block(p.gu, j, 2 * n0) + (s & 1) * kHalf;
          q.b[1] = q.b[0] + kBlock3;
          q.b_pieces = q.n > 64 ? 2 : 1, q.b_mn = true;
        } else {
          q.b[0] = block(p.d, n0, j), q.b[1] = q.b[0] + kHalf;
          q.b_pieces = q.n > 64 ? 2 : 1, q.b_mn = false;
        }
      } else {
        q.a[0] = block(second ? p.dy : p.x, m, c);
        k = (second ? p.dout : p.din) - c * kStep;
        if (second) {  // Wd's rows (O) of the chunk's columns
          q.b[0] = block(p.d, c >> 1, n0) + (c & 1) * kHalf, q.b[1] = nullptr;
          q.b_pieces = 1, q.b_mn = true, q.n = 64;
        } else {
          q.b[0] = block(p.gu, n0, c), q.b[1] = q.b[0] + kHalf;
          q.b_pieces = 2, q.b_mn = false;
        }
      }
      q.a[1] = q.a[0] + kHalf, q.a_pieces = 2;
      q.steps = min(4, (k + 15) >> 4);
    }
    return q;
  }
};

template <int kJob>
__global__ void __launch_bounds__(kThreads32) ffn_tc32_kernel(const __grid_constant__ Tc32Params p) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[2], done[2], drained[2];
  __shared__ uint32_t tmem_slot;
  constexpr bool kHid = kJob <= kHiddenBwd;
  constexpr uint32_t kCols = 256;  // two accumulators
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kIssuer = kAdders / 32, kCopier = kIssuer + 1;
  const Tile32<kJob> tile(p);
  const int total = tile.total;

  if (warp == kIssuer) {
    tmem_alloc(&tmem_slot, kCols);
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&full[i], 1), mbar_init(&done[i], 1);
        mbar_init(&drained[i], kAdders / 32);
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

  if (warp < kIssuer) {
    const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const int n = tile.columns();
    // hidden: 32 columns of G, U and dH; else 64 of the tile, in the first four
    constexpr int kSums = kJob == kHiddenBwd ? 6 : 4;
    float sum[kSums][16];
#pragma unroll
    for (int q = 0; q < kSums; ++q)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[q][i] = 0.f;
    auto add = [&](int col, float (&to)[16]) {
      float v[16];
      tmem_ld(acc + quarter + col, v);
      tmem_wait_ld(v);
#pragma unroll
      for (int i = 0; i < 16; ++i) to[i] += v[i];
    };
    for (int s = 0; s < total; ++s) {
      wait(&done[s & 1], s >> 1);
      tc_fence_after();
      const int at = (s & 1) * 128;
      if constexpr (kHid) {
        if (kJob == kHiddenBwd && s >= p.x.col_blocks) {
#pragma unroll
          for (int q = 4; q < kSums; ++q) add(at + 32 * half + 16 * (q - 4), sum[q]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) add(at + 64 * (q >> 1) + 32 * half + 16 * (q & 1), sum[q]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (64 * half + 16 * q < n) add(at + 64 * half + 16 * q, sum[q]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&drained[s & 1]);
    }
    if constexpr (kHid) {
      // Rows past the last and hidden values past H come out as zeros, which
      // the blocks have to hold.
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int u8 = 0; u8 < 2; ++u8) {
          float h[8], dg[8], du[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = sum[q][8 * u8 + i], u = sum[2 + q][8 * u8 + i];
            const float sg = __fdividef(1.f, 1.f + __expf(-x)), act = x * sg;
            h[i] = act * u;
            if constexpr (kJob == kHiddenBwd) {
              const float d = sum[4 + q][8 * u8 + i];
              dg[i] = (sg + act * (1.f - sg)) * u * d;
              du[i] = d * act;
            }
          }
          // The stages' memory is free now: the blocks are put together there
          // (16-byte stores to global memory took four fifths of the kernel).
          const uint32_t at = base + unit_offset(row, 4 * half + 2 * q + u8);
          auto put = [&](int matrix, const float (&v)[8]) {
            split8(v, [&](int part, uint4 w) {
              st_shared16(at + matrix * kBlock3 + part * kPart, w);
            });
          };
          put(0, h);
          if constexpr (kJob == kHiddenBwd) put(1, dg), put(2, du);
        }
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, %0;" ::"n"(kAdders) : "memory");
      if (threadIdx.x == 0) {
        const int64_t block = (static_cast<int64_t>(tile.m) * p.h.col_blocks + tile.n0) * kBlock3;
        const uint8_t* from = raw + (base - smem_addr(raw));
        bulk_s2g(p.h.p + block, from, kBlock3);
        if constexpr (kJob == kHiddenBwd) {
          bulk_s2g(p.dg.p + block, from + kBlock3, kBlock3);
          bulk_s2g(p.du.p + block, from + 2 * kBlock3, kBlock3);
        }
        bulk_commit();
        bulk_wait_all();
      }
    } else {
      float* to;
      int width;
      bool on, fresh = true;
      if constexpr (kJob == kOutput) {
        const int64_t r = static_cast<int64_t>(tile.m) * kTile + row;
        width = p.width, on = r < p.rows, to = p.out + r * width;
      } else {
        const int64_t hid = static_cast<int64_t>(tile.m) * kTile + row;
        const int64_t hd = static_cast<int64_t>(p.hid) * p.din;
        width = tile.which < 2 ? p.din : p.dout, on = hid < p.hid, fresh = p.first;
        to = p.out + blockIdx.x * (2 * hd + static_cast<int64_t>(p.hid) * p.dout) + tile.which * hd +
             hid * width;
      }
      const int c0 = tile.n0 * kTile + 64 * half;
      if (on) {
        if (!fresh) {  // all loads before the first store
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (c0 + i < width) sum[i >> 4][i & 15] += to[c0 + i];
        }
        // The output's rows start on 16-byte boundaries where their width allows it;
        // rows of the weights' gradients only if what lies before them in the
        // slices is whole vectors too.
        const bool vec = width % 4 == 0 && aligned16(to);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const float* v = &sum[i >> 4][i & 15];
          if (vec && c0 + i < width) {
            *reinterpret_cast<float4*>(to + c0 + i) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c0 + i + k < width) to[c0 + i + k] = v[k];
          }
        }
      }
    }
  } else if (warp == kIssuer) {
    // Parts of A and B, the smallest products first.
    constexpr int kPa[6] = {0, 1, 2, 0, 1, 0}, kPb[6] = {2, 1, 0, 1, 0, 0};
    constexpr bool kAMn = kJob == kWeights;
    for (int s = 0; s < total; ++s) {
      const int st = s & 1;
      const StagePlan q = tile.stage(s);
      const uint32_t from = base + st * kStage;
      const uint32_t id = tc_idesc(q.n, kAMn, q.b_mn);
      const uint32_t da = kAMn ? desc_mn(from, kHalf) : desc_k(from);
      const uint32_t db = q.b_mn ? desc_mn(from + 3 * kPart, kHalf) : desc_k(from + 3 * kPart);
      const uint32_t sa = kAMn ? kStepMn : kStepK, sb = q.b_mn ? kStepMn : kStepK;
      if (s >= 2) wait(&drained[st], (s >> 1) - 1);
      wait(&full[st], s >> 1);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 6; ++i)
        tc_mma_steps<4>(acc + st * 128, da + kPa[i] * (kPart >> 4), sa, db + kPb[i] * (kPart >> 4), sb,
                        id, q.steps, i > 0);
      tc_commit(&done[st]);
    }
    if (total > 0) wait(&done[(total - 1) & 1], (total - 1) >> 1);
  } else if (warp == kCopier && lane == 0) {
    int s = 0;
    for (; s < total && ok; ++s) {
      const int st = s & 1;
      const StagePlan q = tile.stage(s);
      if (s >= 2) wait(&done[st], (s >> 1) - 1);
      if (!ok) break;
      mbar_arrive_expect_tx(&full[st], 3 * kHalf * (q.a_pieces + q.b_pieces));
      uint8_t* to = raw + (base - smem_addr(raw)) + st * kStage;
      for (int part = 0; part < 3; ++part) {
        for (int i = 0; i < q.a_pieces; ++i)
          bulk_g2s(to + part * kPart + i * kHalf, q.a[i] + part * kPart, kHalf, &full[st]);
        for (int i = 0; i < q.b_pieces; ++i)
          bulk_g2s(to + (3 + part) * kPart + i * kHalf, q.b[i] + part * kPart, kHalf, &full[st]);
      }
    }
    if (!ok)  // copies in flight land before the block leaves
      for (int i = max(0, s - 2); i < s; ++i) tc_wait(&full[i & 1], (i >> 1) & 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_free(acc, kCols);
  }
}

template <int kJob>
int launch32(const Tc32Params& p, dim3 grid, cudaStream_t s) {
  const int smem = 2 * kStage + 1024;
  TGS_CUDA(cudaFuncSetAttribute(ffn_tc32_kernel<kJob>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                smem));
  ffn_tc32_kernel<kJob><<<grid, kThreads32, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

int split(const void* first, const void* second, int64_t ld, int64_t rows, int cols, const Split& to,
          cudaStream_t s) {
  const int64_t tiles = ceil_div<int64_t>(rows, second ? 64 : kTile);
  split_kernel<<<static_cast<unsigned>(tiles * to.col_blocks), 256, 0, s>>>(
      static_cast<const float*>(first), static_cast<const float*>(second), ld, rows, cols, to);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

int blocks64(int w) { return ceil_div(w, 64); }

// Tiles of a batch: its split matrices together take at most about 64 MB of the
// 126 MB of L2; batches of one size.
int64_t batch_tiles(int64_t n, int d, int h, int o, bool backward) {
  const int64_t tiles = ceil_div<int64_t>(n, kTile);
  const int64_t per_tile =
      backward ? blocks64(d) + blocks64(o) + 3 * blocks64(h) : blocks64(d) + blocks64(h);
  const int64_t most = std::max<int64_t>(1, (64ll << 20) / (per_tile * kBlock3));
  return ceil_div(tiles, ceil_div(tiles, most));
}

int weight_tiles(int d, int h, int o) {
  return ceil_div(h, kTile) * (2 * ceil_div(d, kTile) + ceil_div(o, kTile));
}

int64_t partial_floats(int64_t n, int d, int h, int o) {
  return ceil_div<int64_t>(tc32_slices(n, d, h, o) * static_cast<int64_t>(h) * (2 * d + o), 4) * 4;
}

}  // namespace

int tc32_slices(int64_t n, int d, int h, int o) {
  const int64_t halves = 2 * batch_tiles(n, d, h, o, true);
  const int64_t most = std::max(1, 2 * sm_count() / weight_tiles(d, h, o));
  return static_cast<int>(std::min<int64_t>(most, ceil_div<int64_t>(halves, 8)));
}

int64_t tc32_scratch_floats(int64_t n, int d, int h, int o, bool backward) {
  const int64_t weights = static_cast<int64_t>(blocks64(h)) * (blocks64(d) + ceil_div(o, kTile));
  const int64_t tiles = batch_tiles(n, d, h, o, backward);
  const int64_t per_tile =
      backward ? blocks64(d) + blocks64(o) + 3 * blocks64(h) : blocks64(d) + blocks64(h);
  return (weights + tiles * per_tile) * (kBlock3 / 4) + (backward ? partial_floats(n, d, h, o) : 0);
}

int ffn_tc32_run(const FfnParams& f, bool backward, cudaStream_t s) {
  const int64_t batch = batch_tiles(f.n, f.d, f.h, f.o, backward);
  const int slices = backward ? tc32_slices(f.n, f.d, f.h, f.o) : 0;
  const bool weights = backward && f.dwg;
  uint8_t* next = reinterpret_cast<uint8_t*>(f.scratch + (backward ? partial_floats(f.n, f.d, f.h, f.o) : 0));
  auto take = [&](int64_t row_tiles, int col_blocks) {
    const Split t{next, col_blocks};
    next += row_tiles * col_blocks * kBlock3;
    return t;
  };
  Tc32Params p{};
  p.hid = f.h, p.din = f.d, p.dout = f.o, p.bwd = backward, p.err = f.err;
  p.width = backward ? f.d : f.o;
  p.gu = take(blocks64(f.h), blocks64(f.d));
  p.d = take(ceil_div(f.o, kTile), blocks64(f.h));
  p.x = take(batch, blocks64(f.d));
  p.h = take(batch, blocks64(f.h));
  if (backward) {
    p.dy = take(batch, blocks64(f.o));
    p.dg = take(batch, blocks64(f.h)), p.du = take(batch, blocks64(f.h));
  }
  if (int rc = split(f.wg, f.wu, f.d, f.h, f.d, p.gu, s)) return rc;
  if (int rc = split(f.wd, nullptr, f.h, f.o, f.h, p.d, s)) return rc;
  for (int64_t r0 = 0; r0 < f.n; r0 += batch * kTile) {
    p.rows = std::min(batch * kTile, f.n - r0);
    p.tiles = static_cast<int>(ceil_div<int64_t>(p.rows, kTile));
    if (int rc = split(static_cast<const float*>(f.x) + r0 * f.x_stride, nullptr, f.x_stride, p.rows,
                       f.d, p.x, s))
      return rc;
    const dim3 hidden(p.tiles, blocks64(f.h));
    if (backward) {
      if (int rc = split(static_cast<const float*>(f.dy) + r0 * f.dy_stride, nullptr, f.dy_stride,
                         p.rows, f.o, p.dy, s))
        return rc;
      if (int rc = launch32<kHiddenBwd>(p, hidden, s)) return rc;
    } else if (int rc = launch32<kHidden>(p, hidden, s)) {
      return rc;
    }
    if (f.y) {
      p.out = static_cast<float*>(f.y) + r0 * p.width;
      if (int rc = launch32<kOutput>(p, dim3(p.tiles, ceil_div(p.width, kTile)), s)) return rc;
    }
    if (weights) {
      p.out = f.scratch;
      p.per_slice = ceil_div(2 * p.tiles, slices);
      p.first = r0 == 0;
      if (int rc = launch32<kWeights>(p, dim3(slices, weight_tiles(f.d, f.h, f.o)), s)) return rc;
    }
  }
  return TGS_OK;
}

}  // namespace tgs
