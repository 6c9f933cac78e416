// Gated feed-forward block in bf16 on the 5th-generation tensor cores; the
// formulas stand in tgs_ffn.cu.
//
// One persistent block per SM takes tiles of 128 rows. Per chunk of 64 hidden
// values, "first" products (G and U as one N = 128 product; in the backward
// dH too) land in tensor memory, eight warps turn them into the hidden chunk
// (backward: dG and dU), rounded to bf16 into shared memory, and "second"
// products add that chunk's share to the output tile's accumulators (Y, or
// dX). The roles are warps of their own joined by mbarriers, so loads,
// products and the activation of different chunks run at once:
//   warps 0-15   activation: two groups of eight take turns by chunk
//   warps 16, 17 issue the first and the second products (a warp each: the
//                next chunk's first products do not wait behind the output)
//   warp  18     weight blocks (bulk copies)
//   warp  19     row tiles by tensor-map copies
//   warps 20-23  the output tile
// The same block of weights serves both products: as K-major operand of one
// and as MN-major operand of the other.
//
// Rounding the hidden values to bf16 adds as much error to the results as
// rounding those does, 0.0024 of a result in place of 0.0017. The forward keeps
// them in two bf16 parts (kFine), for 5 to 12 % of its time, so that a row's
// output is 0.0017 off and the same in calls of any size. In the backward two
// parts take up to twice as long (2,097,152 rows of 64 -> 128 -> 48: 830 us
// against 400; 1,500 of 256 -> 4096 -> 256: 645 against 370; 1,500 of 32 -> 64
// -> 3: 127 against 122, most of it the host's), so calls of up to kFineRows
// rows have them and larger ones keep one part.
//
// Bound: at 64 -> 128 -> 48 the special-function unit (65 % busy) and waits
// between the roles: 2,097,152 rows forward 192 us (2.4 TB/s), backward in one
// kernel 400 us; at 256 -> 512 -> 256 the matrix instructions (a third of the
// forward's are those of the second parts): 400,000 rows forward 359 us, 0.88
// PFLOP/s of the block's own products, 52 % of the measured rate.
//
// Weights stay in shared memory where they fit (then the blocks lay them out
// themselves); else a small kernel lays them out once per call and they
// stream through a ring of 16 KB slots, out of L2.
#include <cuda_bf16.h>

#include <atomic>

#include "tgs_ffn.cuh"
#include "tgs_tc.cuh"

namespace tgs {
namespace {

constexpr int kEpi = 512;      // activation threads, in two groups
constexpr int kOut = 128;      // threads of the output
constexpr int kTcThreads = kEpi + 128 + kOut;
constexpr int kWarpF = kEpi / 32, kWarpS = kWarpF + 1, kWarpW = kWarpF + 2, kWarpT = kWarpF + 3;
constexpr int kTile = 128;     // rows
constexpr int kChunk = 64;     // hidden values
constexpr int kMaxTiles = 3;   // row-tile buffers
constexpr int kMaxHid = 4;     // hidden buffers
constexpr int kMaxSlots = 12;  // weight ring
// Tiles whose products the accumulators of the weights' gradients take up before
// they are added to the block's sums in memory (128: 1,024 instructions, twice
// that with kFine). An instruction cuts off, always towards zero, what does not
// fit the sum's 24 bits: over 300,000 rows of one slice, products of one sign
// lost 1.8e-3 of the gradient without an end to it, 1.7e-4 with one every 256
// tiles, 7e-5 every 128, 2e-5 every 64, where its own rounding to bf16 is 1.7e-3.
// Every 64 costs 13 of 183 us at 200,001 rows of 128 -> 384 -> 128, every 128 none.
constexpr int kSweep = 128;
// Rows of a call whose backward keeps hidden values in two parts: a tile for
// each SM of a B200, but the same number everywhere.
constexpr int kFineRows = 148 * kTile;
constexpr int kSmemBudget = 227 * 1024 - 2048;  // less alignment and barriers

struct TcParams {
  CUtensorMap xmap, dymap;
  FfnParams f;
  const uint8_t* packed;  // laid-out weights (streaming)
  float* partial;         // the weights' gradients by slice
  int64_t tiles;
  int cd, co, nc;  // operand blocks of D and O, chunks of H
  int kd, ko;      // 16-steps of D and O
  int nx, nh, nb, ny, slots, slots_f;  // buffers: row tiles, hidden, first and output accumulators
  int ycols;                  // columns of one output accumulator
  int resident, vec_y, fine;
  uint32_t tile_bytes, h_bytes, w_bytes, stage_bytes;
  uint32_t tmem_cols;
  // Block b takes chunks [cpc g, cpc g + cpc) of tiles s, s + slices, ... with
  // g = b % groups and s = b / groups. With `split`, odd g are the blocks of
  // dWd's gradient and even g those of the two others (for chunks g / 2).
  int cpc, groups, slices, split;
};

// What a kernel computes: Y, dX, the weights' gradients, or the last two.
enum : int { kFwd = 0, kDx = 1, kDw = 2, kDxDw = 3 };

struct TcBars {
  uint64_t xfull[kMaxTiles], xempty[kMaxTiles];
  uint64_t gfull[2], gempty[2], hfull[kMaxHid], hempty[kMaxHid];
  uint64_t yfull[2], yempty[2], done, accfull, accempty;
  uint64_t wfull[kMaxSlots], wempty[kMaxSlots];
  uint32_t tmem;
};

// --- weights in operand layout -------------------------------------------------
// Per chunk j: cd blocks [128][64] of D's columns, rows 0-63 the chunk's rows
// of Wg and rows 64-127 those of Wu; then (after all chunks' blocks) Wd's
// columns of the chunk as [16 ko][64]. Zeros beyond D, H and O.

// `nj` chunks are laid out.
__host__ __device__ __forceinline__ uint32_t wgu_offset(const TcParams& p, int j, int c) {
  return static_cast<uint32_t>(j * p.cd + c) * kBlockBytes;
}
__host__ __device__ __forceinline__ uint32_t wd_offset(const TcParams& p, int nj, int j, int b) {
  return static_cast<uint32_t>(nj * p.cd) * kBlockBytes + j * p.ko * 2048 + b * kBlockBytes;
}
__host__ __device__ __forceinline__ uint32_t weight_bytes(const TcParams& p, int nj) {
  return static_cast<uint32_t>(nj) * (p.cd * kBlockBytes + p.ko * 2048);
}

__device__ __forceinline__ uint4 load_unit(const __nv_bfloat16* src, int64_t at, int left,
                                           bool vec) {
  if (left >= 8 && vec) return *reinterpret_cast<const uint4*>(src + at);
  union {
    uint4 q;
    uint16_t t[8];
  } u;
  u.q = make_uint4(0, 0, 0, 0);
  const uint16_t* s = reinterpret_cast<const uint16_t*>(src) + at;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) u.t[i] = s[i];
  return u.q;
}

// 16-byte unit `e` of the layout of chunks j0 to j0 + nj: its value, and
// where it goes.
__device__ __forceinline__ uint4 weight_unit(const TcParams& p, int j0, int nj, uint32_t e,
                                             uint32_t* offset) {
  const FfnParams& f = p.f;
  const uint32_t block = e >> 10, gu_blocks = nj * p.cd;
  if (block < gu_blocks) {
    const int j = block / p.cd, c = block - j * p.cd;
    const int row = (e >> 3) & 127, unit = e & 7;
    const int hid = (j0 + j) * kChunk + (row & 63), col = c * kBlockCols + unit * 8;
    *offset = block * kBlockBytes + unit_offset(row, unit);
    if (hid >= f.h || col >= f.d) return make_uint4(0, 0, 0, 0);
    const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(row < 64 ? f.wg : f.wu);
    const bool vec = f.d % 8 == 0 && aligned16(w);
    return load_unit(w, static_cast<int64_t>(hid) * f.d + col, f.d - col, vec);
  }
  const uint32_t r = (e - (gu_blocks << 10)) >> 3;  // row over all chunks
  const int j = r / (16 * p.ko), row = r - j * 16 * p.ko, unit = e & 7;
  const int col = (j0 + j) * kChunk + unit * 8;
  *offset = gu_blocks * kBlockBytes + j * p.ko * 2048 + unit_offset(row, unit);
  if (row >= f.o || col >= f.h) return make_uint4(0, 0, 0, 0);
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(f.wd);
  const bool vec = f.h % 8 == 0 && aligned16(w);
  return load_unit(w, static_cast<int64_t>(row) * f.h + col, f.h - col, vec);
}

__global__ void __launch_bounds__(256) ffn_pack_kernel(const TcParams p, uint8_t* dst) {
  const uint32_t e = blockIdx.x * 256 + threadIdx.x;
  if (e >= weight_bytes(p, p.nc) / 16) return;
  uint32_t at;
  const uint4 v = weight_unit(p, 0, p.nc, e, &at);
  *reinterpret_cast<uint4*>(dst + at) = v;
}

// Rows of 16-bit values to rows of whole 16-byte units, zeros at their ends.
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ src,
                                                         int64_t stride, int64_t n, int c,
                                                         uint4* __restrict__ dst, int units) {
  const int64_t all = n * units;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < all;
       e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / units;
    const int col = static_cast<int>(e - row * units) * 8;
    const uint16_t* s = src + row * stride + col;
    union {
      uint4 q;
      uint16_t t[8];
    } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.t[i] = col + i < c ? s[i] : 0;
    dst[e] = u.q;
  }
}

// --- waits -----------------------------------------------------------------------
// Every wait has a limit. After one has run out, the thread records it, skips
// its later waits and leaves with the others; the outputs are then undefined.
struct Waits {
  int32_t* err;
  bool ok = true;
  __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t phase) {
    if (ok && !tc_wait(bar, phase & 1)) {
      ok = false;
      report_error(err, TGS_DEV_WAIT_TIMEOUT, blockIdx.x, threadIdx.x);
    }
  }
};

// One arrival for the warp, after all of its lanes have come here (an arrival of
// each thread takes the same time: 168 us for either, forward of 2,097,152 rows
// of 64 -> 128 -> 48).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// --- activation --------------------------------------------------------------------
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 + exp(-g) of two values.
__device__ __forceinline__ F2 one_plus_exp(F2 g) {
  float ea, eb;
  (g * F2(-1.4426950408889634f, -1.4426950408889634f)).get(ea, eb);
  return F2(fast_exp2(ea), fast_exp2(eb)) + F2(1.f, 1.f);
}

// Two values rounded and packed; with kFine also what the rounding left, in a
// second bf16 part.
template <bool kFine>
__device__ __forceinline__ void round_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(a, b);
  if constexpr (kFine)
    lo = pack_bf16(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

// silu(g) u = g / (1 + exp(-g)) u of kW values, rounded and packed in pairs. The
// gate comes first: a closed one gives 0 however large g u is.
// The special-function unit (16 results a cycle and SM) takes two operations a
// value. One reciprocal for two values, 1 / a = b / (a b), saves a quarter of
// them but costs as much again in products and moves: 196 against 168 us for
// 2,097,152 rows of 64 -> 128 -> 48 with hidden values of one part, and 168 with
// it for every second pair.
template <int kW>
__device__ __forceinline__ void gate(const float (&g)[kW], const float (&u)[kW],
                                     uint32_t (&h)[kW / 2], uint32_t (&lo)[kW / 2]) {
#pragma unroll
  for (int i = 0; i < kW; i += 2) {
    const F2 g2(g[i], g[i + 1]);
    float a, b;
    one_plus_exp(g2).get(a, b);
    (g2 * F2(fast_rcp(a), fast_rcp(b)) * F2(u[i], u[i + 1])).get(a, b);
    round_pair<true>(a, b, h[i / 2], lo[i / 2]);
  }
}

// The backward's hidden values, rounded and packed in pairs: dG, dU, and (for
// the weights' gradients) h.
template <bool kH, bool kFine, int kW>
__device__ __forceinline__ void gate_backward(const float (&g)[kW], const float (&u)[kW],
                                              const float (&dh)[kW], uint32_t (&h)[kW / 2],
                                              uint32_t (&dg)[kW / 2], uint32_t (&du)[kW / 2],
                                              uint32_t (&h_lo)[kW / 2], uint32_t (&dg_lo)[kW / 2],
                                              uint32_t (&du_lo)[kW / 2]) {
#pragma unroll
  for (int i = 0; i < kW; i += 2) {
    const F2 g2(g[i], g[i + 1]), u2(u[i], u[i + 1]), d2(dh[i], dh[i + 1]);
    float a, b;
    one_plus_exp(g2).get(a, b);
    // s dh first: a closed gate gives 0 however large dh u is. silu'(g) =
    // s (1 + g (1 - s)).
    const F2 s2(fast_rcp(a), fast_rcp(b)), sd = s2 * d2;
    const F2 slope = fma2(g2, fma2(s2, F2(-1.f, -1.f), F2(1.f, 1.f)), F2(1.f, 1.f));
    if constexpr (kH) {
      (g2 * s2 * u2).get(a, b);
      round_pair<kFine>(a, b, h[i / 2], h_lo[i / 2]);
    }
    (sd * u2 * slope).get(a, b);
    round_pair<kFine>(a, b, dg[i / 2], dg_lo[i / 2]);
    (g2 * sd).get(a, b);
    round_pair<kFine>(a, b, du[i / 2], du_lo[i / 2]);
  }
}

// Puts kW values into a block's row, from column kW g on.
template <int kN>
__device__ __forceinline__ void store_granule(uint32_t block, uint32_t row, uint32_t g,
                                              const uint32_t (&v)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / 4; ++i)
    st_shared16(block + unit_offset(row, g * (kN / 4) + i),
                make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
}

// The output tile's row `lane_row`, out of its accumulators. A tile of the
// output is one piece of memory that starts on a 16-byte boundary; where its
// rows do not, it is put together at `stage` and stored as a whole (2-byte
// stores of rows of 59 took three times the kernel's other work). `stage` 0:
// the rows are stored apart (aligned ones, or no room).
__device__ __forceinline__ void store_output(const TcParams& p, uint32_t acc, int64_t tile,
                                             int out, int lane_row, uint32_t stage) {
  __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.f.y);
  const int64_t row = tile * kTile + lane_row;
  for (int c = 0; c < out; c += 16) {
    float v[16];
    tmem_ld(acc + c, v);
    tmem_wait_ld(v);
    __nv_bfloat16* dst = y + row * out + c;
    if (stage) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < out)
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(stage + 2 * (lane_row * out + c + i)),
                       "h"(__bfloat16_as_ushort(__float2bfloat16_rn(v[i])))
                       : "memory");
    } else if (row >= p.f.n) {
    } else if (p.vec_y) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (c + 8 * u < out) {
          uint4 q;
          q.x = pack_bf16(v[8 * u + 0], v[8 * u + 1]);
          q.y = pack_bf16(v[8 * u + 2], v[8 * u + 3]);
          q.z = pack_bf16(v[8 * u + 4], v[8 * u + 5]);
          q.w = pack_bf16(v[8 * u + 6], v[8 * u + 7]);
          *reinterpret_cast<uint4*>(dst + 8 * u) = q;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < out) dst[i] = __float2bfloat16_rn(v[i]);
    }
    __syncwarp();  // the next load is the whole warp's
  }
}

// The staged tile, by the output's threads.
__device__ __forceinline__ void store_staged(const TcParams& p, int64_t tile, int out,
                                             const uint8_t* stage, int tid) {
  asm volatile("bar.sync 1, %0;" ::"n"(kOut) : "memory");
  const int64_t left = p.f.n - tile * kTile;
  const int bytes = static_cast<int>(left < kTile ? left : kTile) * out * 2;
  uint8_t* y = static_cast<uint8_t*>(p.f.y) + tile * kTile * out * 2;
  for (int e = tid; e < bytes / 16; e += kOut)
    reinterpret_cast<uint4*>(y)[e] = reinterpret_cast<const uint4*>(stage)[e];
  for (int e = (bytes & ~15) / 2 + tid; e < bytes / 2; e += kOut)
    reinterpret_cast<uint16_t*>(y)[e] = reinterpret_cast<const uint16_t*>(stage)[e];
  asm volatile("bar.sync 1, %0;" ::"n"(kOut) : "memory");
}

// One weight gradient's chunk, out of its accumulators: the block's sum in
// memory, or (`add`) a further share of it.
__device__ __forceinline__ void store_partial(uint32_t acc, float* dst, int cols, bool on, bool add) {
  for (int c = 0; c < cols; c += 16) {
    float v[16];
    tmem_ld(acc + c, v);
    tmem_wait_ld(v);
    if (on) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        float4* to = reinterpret_cast<float4*>(dst + c + i);
        const float4 s = add ? *to : make_float4(0.f, 0.f, 0.f, 0.f);
        *to = make_float4(s.x + v[i], s.y + v[i + 1], s.z + v[i + 2], s.w + v[i + 3]);
      }
    }
    __syncwarp();
  }
}

// Floats of a chunk's gradients in `partial`: [128][16 kd] rows of dWg and
// dWu, then [64][16 ko] columns of dWd.
__host__ __device__ __forceinline__ int chunk_floats(const TcParams& p) {
  return 16 * (128 * p.kd + 64 * p.ko);
}

// --- the kernel --------------------------------------------------------------------
template <int kMode, bool kFine>
__global__ void __launch_bounds__(kTcThreads, 1) ffn_tc_kernel(const __grid_constant__ TcParams p) {
  extern __shared__ uint8_t raw[];
  __shared__ TcBars bars;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t xs = base;                             // nx tiles: X blocks, then dY blocks
  const uint32_t hs = xs + p.nx * p.tile_bytes;         // nh hidden buffers
  const uint32_t ws = hs + p.nh * p.h_bytes;            // weights, or the ring
  const uint32_t ys = ws + (p.resident ? p.w_bytes : p.slots * kBlockBytes);  // staged output
  // from lane 0, so that the compiler sees the roles' branches as uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr bool kBwd = kMode != kFwd, kHasDw = kMode >= kDw, kRows = kMode != kDw;
  // second parts in a hidden buffer
  const uint32_t lo_at = (!kBwd ? 1 : kHasDw && !p.split ? 3 : 2) * kBlockBytes;
  const int group_id = kHasDw ? blockIdx.x % p.groups : 0;
  const int slice = kHasDw ? blockIdx.x / p.groups : blockIdx.x;
  const bool want_gu = !kHasDw || !p.split || !(group_id & 1);  // dWg and dWu
  const bool want_d = !kHasDw || !p.split || (group_id & 1);    // dWd
  const int j0 = (p.split ? group_id >> 1 : group_id) * p.cpc;
  const int nj = min(p.cpc, p.nc - j0);
  const int mine = static_cast<int>((p.tiles - slice + p.slices - 1) / p.slices);
  const int steps = mine * nj;  // n <= 2^31 and H <= 4096: below 2^30 of them
  // where chunk j's weights are: of this block's chunks, or of all
  const int laid = p.resident ? p.cpc : p.nc, jw = p.resident ? 0 : j0;
  const int wblocks = (p.ko + 7) / 8;  // blocks of Wd per chunk
  constexpr uint32_t kGCols = kBwd ? 192 : 128;
  Waits wait{p.f.err};

  if (warp == kWarpF) {
    tmem_alloc(&bars.tmem, p.tmem_cols);
    if (lane == 0) {
      for (int i = 0; i < kMaxTiles; ++i) mbar_init(&bars.xfull[i], 1), mbar_init(&bars.xempty[i], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&bars.gfull[i], 1), mbar_init(&bars.gempty[i], kEpi / 64);
        mbar_init(&bars.yfull[i], 1), mbar_init(&bars.yempty[i], kOut / 32);
      }
      for (int i = 0; i < kMaxHid; ++i) mbar_init(&bars.hfull[i], kEpi / 64), mbar_init(&bars.hempty[i], 1);
      mbar_init(&bars.done, 2), mbar_init(&bars.accfull, 1), mbar_init(&bars.accempty, kOut / 32);
      for (int i = 0; i < kMaxSlots; ++i) mbar_init(&bars.wfull[i], 1), mbar_init(&bars.wempty[i], 1);
      fence_mbar_init();
    }
  }
  if (p.resident) {
    for (uint32_t e = threadIdx.x; e < p.w_bytes / 16; e += kTcThreads) {
      uint32_t at;
      const uint4 v = weight_unit(p, j0, p.cpc, e, &at);
      st_shared16(ws + at, v);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  const uint32_t yacc = tmem + p.nb * kGCols;
  const uint32_t wacc = yacc + p.ny * p.ycols;  // gradients: per chunk gu_cols + d_cols
  const uint32_t gu_cols = want_gu ? 16 * p.kd : 0, d_cols = want_d ? 16 * p.ko : 0;
  const uint32_t dg_at = kHasDw && want_d ? kBlockBytes : 0;  // hidden buffer: h, dG, dU

  // Step `it` (tile it / nj, chunk it % nj) signals on the barriers it % 2, and
  // it % hm for the hidden buffers, a tile t on those of t % 2, whether or not
  // there are two buffers: a wait then never meets a barrier that is two phases
  // from the awaited one, which it could not tell from it.
  const int hm = max(p.nh, 2);
  if (warp < kWarpF) {
    // Activation: group warp / 8 takes the steps of its parity; this thread's
    // row of the tile, and every second granule of kW columns of the chunk.
    const uint32_t row = (warp & 3) * 32 + lane;
    const int group = warp >> 3, half = warp >> 2 & 1;
    const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;  // lane 32 (warp % 4)
    int j = group;
    int hb = group, hphase = 0;
    for (int it = group; it < steps; it += 2, j += 2, hb += 2) {
      while (j >= nj) j -= nj;
      if (hb >= hm) hb -= hm, ++hphase;
      wait(&bars.gfull[group], it >> 1);
      tc_fence_after();
      const uint32_t acc = tmem + (p.nb == 2 ? group : 0) * kGCols + quarter;
      const uint32_t hbuf = hs + (p.nh > 1 ? hb : 0) * p.h_bytes;
      // whole 16-steps of the chunk's hidden values
      const int cols = (min(kChunk, p.f.h - (j0 + j) * kChunk) + 15) & ~15;
      constexpr int kParts = kBwd ? 3 : 2;  // G, U, dH
      constexpr int kW = kHasDw || (kFine && kBwd) ? 8 : 16;  // what the registers hold
      constexpr int kTurns = kChunk / kW / 2;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int q = half + 2 * i;
        float v[kParts][kW];
        if (q * kW < cols) {
#pragma unroll
          for (int k = 0; k < kParts; ++k) tmem_ld(acc + 64 * k + kW * q, v[k]);
        }
        if (i == 0) {  // meanwhile: the step that last used the hidden buffer
          if (p.nh > 1) {
            if (hphase > 0) wait(&bars.hempty[hb], hphase - 1);
          } else if (it > 0) {
            wait(&bars.hempty[(it - 1) & 1], (it - 1) >> 1);
          }
        }
        if (q * kW < cols) {
#pragma unroll
          for (int k = 0; k < kParts; ++k) tmem_wait_ld(v[k]);
        }
        if (i == kTurns - 1) {
          tc_fence_before();
          warp_arrive(&bars.gempty[group], lane);  // the accumulators have been read
        }
        if (q * kW < cols) {
          uint32_t h[kW / 2], dg[kW / 2], du[kW / 2];
          uint32_t h_lo[kW / 2], dg_lo[kW / 2], du_lo[kW / 2];
          if constexpr (kBwd) {
            gate_backward<kHasDw, kFine>(v[0], v[1], v[kParts - 1], h, dg, du, h_lo, dg_lo, du_lo);
          } else {
            gate(v[0], v[1], h, h_lo);
          }
          if (kMode == kFwd || (kHasDw && want_d)) store_granule(hbuf, row, q, h);
          if (kBwd && want_gu) {
            store_granule(hbuf + dg_at, row, q, dg);
            store_granule(hbuf + dg_at + kBlockBytes, row, q, du);
          }
          if constexpr (kFine) {
            if (kMode == kFwd || (kHasDw && want_d)) store_granule(hbuf + lo_at, row, q, h_lo);
            if (kBwd && want_gu) {
              store_granule(hbuf + lo_at + dg_at, row, q, dg_lo);
              store_granule(hbuf + lo_at + dg_at + kBlockBytes, row, q, du_lo);
            }
          }
        }
      }
      fence_proxy_async_smem();
      warp_arrive(&bars.hfull[hb], lane);
    }
  } else if (warp == kWarpF || warp == kWarpS) {
    // Each warp has a ring of its own (of one ring, each would miss phases).
    const int ring = warp == kWarpF ? 0 : p.slots_f;
    const int ring_end = warp == kWarpF ? p.slots_f : p.slots;
    int slot = ring, wround = 0;
    auto acquire = [&](uint32_t fixed) {
      if (p.resident) return ws + fixed;
      wait(&bars.wfull[slot], wround);
      return ws + slot * kBlockBytes;
    };
    auto release = [&] {
      if (p.resident) return;
      tc_commit(&bars.wempty[slot]);
      if (++slot == ring_end) slot = ring, ++wround;
    };
    if (warp == kWarpF) {
      int j = 0, xb = 0, xround = 0;
      for (int it = 0; it < steps; ++it) {
        const uint32_t x = xs + xb * p.tile_bytes, dy = x + p.cd * kBlockBytes;
        const uint32_t acc = tmem + (p.nb == 2 ? it & 1 : 0) * kGCols;
        if (j == 0) wait(&bars.xfull[xb], xround);
        const int before = it - p.nb;
        if (before >= 0) wait(&bars.gempty[before & 1], before >> 1);
        tc_fence_after();
        for (int c = 0; c < p.cd; ++c) {
          const uint32_t w = acquire(wgu_offset(p, j, c));
          tc_mma_steps<4>(acc, desc_k(x + c * kBlockBytes), kStepK, desc_k(w), kStepK,
                          tc_idesc(128, false, false), p.kd - 4 * c, c > 0);
          release();
        }
        if constexpr (kBwd) {
          for (int b8 = 0; b8 < wblocks; ++b8) {
            const uint32_t w = acquire(wd_offset(p, laid, j, b8));
            for (int c = 0; c < 2 && 2 * b8 + c < p.co; ++c)
              tc_mma_steps<4>(acc + 128, desc_k(dy + (2 * b8 + c) * kBlockBytes), kStepK,
                              desc_mn(w + c * 64 * 128, kBlockBytes), kStepMn,
                              tc_idesc(64, false, true), p.ko - 8 * b8 - 4 * c, b8 + c > 0);
            release();
          }
        }
        tc_commit(&bars.gfull[it & 1]);
        if (++j == nj) {
          if (!kHasDw) tc_commit(&bars.xempty[xb]);
          j = 0;
          if (++xb == p.nx) xb = 0, ++xround;
        }
      }
    } else {
      int j = 0, t = 0, hb = 0, hphase = 0, xb = 0;
      int left = kSweep;  // tiles of the gradients' sweep to come
      for (int it = 0; it < steps; ++it) {
        wait(&bars.hfull[hb], hphase);
        if (kRows && j == 0 && t >= p.ny) wait(&bars.yempty[(t - p.ny) & 1], (t - p.ny) >> 1);
        if (kHasDw && left == 0) {
          wait(&bars.accempty, t / kSweep - 1);
          left = kSweep;
        }
        tc_fence_after();
        const uint32_t y = yacc + (p.ny == 2 ? t & 1 : 0) * p.ycols;
        const uint32_t h = hs + (p.nh > 1 ? hb : 0) * p.h_bytes;
        const int ks = (min(kChunk, p.f.h - (j0 + j) * kChunk) + 15) >> 4;
        if constexpr (kHasDw) {
          // Operands with rows as K: [dG | dU]^T X as one product of 128 hidden
          // columns; of [h | dG]^T dY only the first 64 are read.
          const uint32_t x = xs + xb * p.tile_bytes, dy = x + p.cd * kBlockBytes;
          const uint32_t acc = wacc + j * (gu_cols + d_cols);
          for (int part = 0; part < (kFine ? 2 : 1); ++part) {
            const uint32_t from = h + part * lo_at;
            if (want_gu)
              tc_mma_steps<8>(acc, desc_mn(from + dg_at, kBlockBytes), kStepMn,
                              desc_mn(x, kBlockBytes), kStepMn, tc_idesc(gu_cols, true, true), 8,
                              left < kSweep || part > 0);
            if (want_d)
              tc_mma_steps<8>(acc + gu_cols, desc_mn(from, kBlockBytes), kStepMn,
                              desc_mn(dy, kBlockBytes), kStepMn, tc_idesc(d_cols, true, true), 8,
                              left < kSweep || part > 0);
          }
        }
        if constexpr (kBwd && kRows) {
          // dG Wg + dU Wu: the blocks' columns are N, their rows K
          const int wide = p.resident ? p.cd : 1;  // neighbouring blocks as one product
          for (int c = 0; c < p.cd; c += wide) {
            const uint32_t w = acquire(wgu_offset(p, j, c));
            const uint32_t id = tc_idesc(min(64 * wide, 16 * p.kd - 64 * c), false, true);
            tc_mma_steps<4>(y + 64 * c, desc_k(h + dg_at), kStepK, desc_mn(w, kBlockBytes), kStepMn,
                            id, ks, j > 0);
            tc_mma_steps<4>(y + 64 * c, desc_k(h + dg_at + kBlockBytes), kStepK,
                            desc_mn(w + 64 * 128, kBlockBytes), kStepMn, id, ks, true);
            if constexpr (kFine) {
              tc_mma_steps<4>(y + 64 * c, desc_k(h + lo_at), kStepK, desc_mn(w, kBlockBytes),
                              kStepMn, id, ks, true);
              tc_mma_steps<4>(y + 64 * c, desc_k(h + lo_at + kBlockBytes), kStepK,
                              desc_mn(w + 64 * 128, kBlockBytes), kStepMn, id, ks, true);
            }
            release();
          }
        }
        if constexpr (!kBwd) {
          const int wide = p.resident ? wblocks : 1;
          for (int b8 = 0; b8 < wblocks; b8 += wide) {
            const uint32_t w = acquire(wd_offset(p, laid, j, b8));
            tc_mma_steps<4>(y + 128 * b8, desc_k(h), kStepK, desc_k(w), kStepK,
                            tc_idesc(min(128 * wide, 16 * p.ko - 128 * b8), false, false), ks,
                            j > 0);
            if constexpr (kFine)
              tc_mma_steps<4>(y + 128 * b8, desc_k(h + lo_at), kStepK, desc_k(w), kStepK,
                              tc_idesc(min(128 * wide, 16 * p.ko - 128 * b8), false, false), ks,
                              true);
            release();
          }
        }
        tc_commit(&bars.hempty[hb]);
        if (++hb == hm) hb = 0, ++hphase;
        if (++j == nj) {
          if (kRows) tc_commit(&bars.yfull[t & 1]);
          if (kHasDw) tc_commit(&bars.xempty[xb]);
          if (kHasDw && (--left == 0 || t + 1 == mine)) tc_commit(&bars.accfull);
          if (++xb == p.nx) xb = 0;
          j = 0, ++t;
        }
      }
    }
    tc_commit(&bars.done);
    if (!tc_wait(&bars.done, 0))
      report_error(p.f.err, TGS_DEV_WAIT_TIMEOUT, blockIdx.x, threadIdx.x);
  } else if (warp == kWarpW) {
    if (lane == 0 && !p.resident) {
      struct Ring {
        int begin, end, slot, round;
      } first{0, p.slots_f, 0, 0}, second{p.slots_f, p.slots, p.slots_f, 0};
      auto put = [&](Ring& r, uint32_t offset, uint32_t bytes) {
        if (r.round > 0) wait(&bars.wempty[r.slot], r.round - 1);
        if (!wait.ok) return;  // after a wait that ran out, no copy may land in a slot in use
        mbar_arrive_expect_tx(&bars.wfull[r.slot], bytes);
        bulk_g2s(raw + (ws - smem_addr(raw)) + r.slot * kBlockBytes, p.packed + offset, bytes,
                 &bars.wfull[r.slot]);
        if (++r.slot == r.end) r.slot = r.begin, ++r.round;
      };
      auto put_gu = [&](Ring& r, int j) {
        for (int c = 0; c < p.cd; ++c) put(r, wgu_offset(p, jw + j, c), kBlockBytes);
      };
      auto put_d = [&](Ring& r, int j) {
        for (int b8 = 0; b8 < wblocks; ++b8)
          put(r, wd_offset(p, laid, jw + j, b8), min(8, p.ko - 8 * b8) * 2048);
      };
      // F0, F1 S0, F2 S1, ...: no first products wait for blocks that only come
      // after those of a second product that waits for them.
      int j1 = 0, j = 0;
      for (int it = -1; it < steps; ++it) {
        if (it + 1 < steps) {
          put_gu(first, j1);
          if (kBwd) put_d(first, j1);
          if (++j1 == nj) j1 = 0;
        }
        if (kRows && it >= 0) {
          if (kBwd) {
            put_gu(second, j);
          } else {
            put_d(second, j);
          }
          if (++j == nj) j = 0;
        }
        if (!wait.ok) break;
      }
      if (!wait.ok) {  // copies in flight land before the block leaves
        for (int i = 0; i < p.slots; ++i) {
          const Ring& g = i < p.slots_f ? first : second;
          const int r = i < g.slot ? g.round : g.round - 1;
          if (r >= 0) tc_wait(&bars.wfull[i], r & 1);
        }
      }
    }
  } else if (warp == kWarpT) {
    if (lane == 0) {
      int xb = 0, round = 0;
      for (int t = 0; t < mine && wait.ok; ++t) {
        if (round > 0) wait(&bars.xempty[xb], round - 1);
        if (!wait.ok) break;
        const int64_t r0 = (slice + static_cast<int64_t>(t) * p.slices) * kTile;
        const uint32_t dst = xs + xb * p.tile_bytes;
        const int xblocks = p.cd, yblocks = kBwd ? p.co : 0;
        mbar_arrive_expect_tx(&bars.xfull[xb], (xblocks + yblocks) * kBlockBytes);
        for (int c = 0; c < xblocks; ++c)
          tma_load_2d(dst + c * kBlockBytes, &p.xmap, c * kBlockCols, static_cast<int>(r0),
                      &bars.xfull[xb]);
        for (int c = 0; c < yblocks; ++c)
          tma_load_2d(dst + (p.cd + c) * kBlockBytes, &p.dymap, c * kBlockCols,
                      static_cast<int>(r0), &bars.xfull[xb]);
        if (++xb == p.nx) xb = 0, ++round;
      }
      if (!wait.ok) {  // copies in flight land before the block leaves
        for (int i = 0; i < p.nx; ++i) {
          const int r = i < xb ? round : round - 1;
          if (r >= 0) tc_wait(&bars.xfull[i], r & 1);
        }
      }
    }
  } else {
    const uint32_t quarter = static_cast<uint32_t>(warp & 3) << 21;
    const int row = (warp & 3) * 32 + lane;
    // The gradients' accumulators at the end of a sweep (at most 1,280 steps).
    auto drain = [&](int sweep) {
      wait(&bars.accfull, sweep);
      tc_fence_after();
      for (int j = 0; j < nj; ++j) {
        float* dst = p.partial + (static_cast<int64_t>(slice) * p.nc + j0 + j) * chunk_floats(p);
        const uint32_t acc = wacc + j * (gu_cols + d_cols) + quarter;
        const bool on = (row & 63) < p.f.h - (j0 + j) * kChunk;
        if (want_gu) store_partial(acc, dst + row * 16 * p.kd, gu_cols, on, sweep > 0);
        if (want_d && row < 64)
          store_partial(acc + gu_cols, dst + 128 * 16 * p.kd + row * 16 * p.ko, d_cols, on, sweep > 0);
      }
      tc_fence_before();
      warp_arrive(&bars.accempty, lane);
    };
    // Output tiles [begin, end).
    auto rows = [&](int begin, int end) {
      const int out = kBwd ? p.f.d : p.f.o;
      for (int t = begin; t < end; ++t) {
        wait(&bars.yfull[t & 1], t >> 1);
        tc_fence_after();
        store_output(p, yacc + (p.ny == 2 ? t & 1 : 0) * p.ycols + quarter,
                     slice + static_cast<int64_t>(t) * p.slices, out, row, p.stage_bytes ? ys : 0);
        tc_fence_before();
        warp_arrive(&bars.yempty[t & 1], lane);
        if (p.stage_bytes)
          store_staged(p, slice + static_cast<int64_t>(t) * p.slices, out, raw + (ys - smem_addr(raw)), row);
      }
    };
    if constexpr (kHasDw) {
      for (int t = 0; t < mine; t += kSweep) {
        if constexpr (kRows) rows(t, min(t + kSweep, mine));
        drain(t / kSweep);
      }
    } else {
      rows(0, mine);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpF) {
    tc_fence_after();
    tmem_free(tmem, p.tmem_cols);
  }
}

// The slices' sums in a fixed order, rounded into the weights' layouts: 128
// neighbouring floats a block, the slices dealt to its eight warps.
__global__ void __launch_bounds__(256) ffn_tc_sum_kernel(const TcParams p) {
  __shared__ float4 part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int floats = chunk_floats(p);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 128 + 4 * lane;
  const int64_t stride = static_cast<int64_t>(p.nc) * floats;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = warp; s < p.slices; s += 8) {
    const float4 v = *reinterpret_cast<const float4*>(p.partial + s * stride + at);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp > 0) return;
  for (int w = 1; w < 8; ++w) {
    const float4 v = part[w][lane];
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
  const int j = static_cast<int>(at / floats), e = static_cast<int>(at - static_cast<int64_t>(j) * floats);
  const FfnParams& f = p.f;
  const int gu = 128 * 16 * p.kd;
  const bool up = e < gu;
  const int width = up ? 16 * p.kd : 16 * p.ko;
  const int row = (up ? e : e - gu) / width, col = (up ? e : e - gu) - row * width;
  const int hid = j * kChunk + (row & 63);
  if (hid >= f.h) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat16 r = __float2bfloat16_rn(v[i]);
    if (up) {
      if (col + i < f.d)
        static_cast<__nv_bfloat16*>(row < 64 ? f.dwg : f.dwu)[static_cast<int64_t>(hid) * f.d + col + i] = r;
    } else if (col + i < f.o) {
      static_cast<__nv_bfloat16*>(f.dwd)[static_cast<int64_t>(col + i) * f.h + hid] = r;
    }
  }
}

uint32_t pow2_cols(uint32_t c) {
  uint32_t p = 32;
  while (p < c) p *= 2;
  return p;
}

TcParams tc_params(const FfnParams& f, bool bwd) {
  TcParams p{};
  p.f = f;
  p.kd = ceil_div(f.d, 16), p.ko = ceil_div(f.o, 16);
  p.cd = ceil_div(f.d, 64), p.co = ceil_div(f.o, 64), p.nc = ceil_div(f.h, kChunk);
  p.tiles = ceil_div<int64_t>(f.n, kTile);
  p.cpc = p.nc, p.groups = 1;
  p.fine = !bwd || f.n <= kFineRows;
  return p;
}

int make_maps(TcParams& p, bool bwd) {
  const FfnParams& f = p.f;
  if (int rc = make_row_map(&p.xmap, f.x, f.n, f.d, f.x_stride)) return rc;
  return bwd ? make_row_map(&p.dymap, f.dy, f.n, f.o, f.dy_stride) : TGS_OK;
}

// Room for a staged output tile, where `least` bytes are left beside it.
void plan_stage(TcParams& p, int out, int64_t least, int64_t& budget) {
  const uint32_t bytes = ceil_div(2 * kTile * out, 1024) * 1024;
  p.stage_bytes = out % 8 != 0 && least + bytes <= budget ? bytes : 0;
  budget -= p.stage_bytes;
}

// Buffers for Y or dX. Shared memory goes first to the weights (as a
// whole where two row tiles and two hidden buffers fit beside them), then to
// whatever keeps the most work in flight.
void plan_rows(TcParams& p, bool bwd) {
  p.tile_bytes = (p.cd + (bwd ? p.co : 0)) * kBlockBytes;
  p.h_bytes = (bwd ? 2 : 1) * (p.fine ? 2 : 1) * kBlockBytes;
  const uint32_t out = bwd ? p.kd * 16 : p.ko * 16, g = bwd ? 192 : 128;
  p.nb = 2 * g + out <= 512 ? 2 : 1;
  p.ny = p.nb * g + 2 * out <= 512 ? 2 : 1;
  p.ycols = out;
  p.tmem_cols = pow2_cols(p.nb * g + p.ny * out);
  p.w_bytes = weight_bytes(p, p.nc);
  p.slices = static_cast<int>(std::min<int64_t>(p.tiles, sm_count()));
  int64_t budget = kSmemBudget;
  plan_stage(p, bwd ? p.f.d : p.f.o, p.tile_bytes + p.h_bytes + 6 * kBlockBytes, budget);
  auto used = [&] { return static_cast<int64_t>(p.nx) * p.tile_bytes + p.nh * p.h_bytes; };
  p.nx = 2, p.nh = 2, p.slots = 1;
  p.resident = used() + p.w_bytes <= budget;
  if (p.resident) {
    for (int nh = kMaxHid; nh >= 2; --nh) {
      p.nh = nh;
      for (p.nx = 3; p.nx >= 2; --p.nx)
        if (used() + p.w_bytes <= budget) return;
    }
  }
  // The rings hold at least one chunk's blocks twice over before a second row
  // tile or hidden buffer is bought with them; they share the slots by the
  // blocks that a step takes from each.
  const int per_chunk = p.cd + (p.ko + 7) / 8;
  for (int more = 3; more >= 0; --more) {
    p.nh = 1 + (more >> 1 & 1), p.nx = 1 + (more & 1);
    p.slots = static_cast<int>(std::min<int64_t>(kMaxSlots, (budget - used()) / kBlockBytes));
    if (p.slots >= std::min(2 * per_chunk, 6)) break;
  }
  const int first = bwd ? per_chunk : p.cd, second = bwd ? p.cd : per_chunk - p.cd;
  p.slots_f = std::min(p.slots - 1, std::max(1, (p.slots * first + (first + second) / 2) / (first + second)));
}

// Buffers for the weights' gradients, whose accumulators stay in tensor memory
// over all of a block's tiles: as many chunks per block as fit there. With
// `dx`, whether all of them fit beside dX's, so that one kernel gives both.
bool plan_weights(TcParams& p, bool dx) {
  const int gu = 16 * p.kd, d = 16 * p.ko;
  p.tile_bytes = (p.cd + p.co) * kBlockBytes;
  p.nb = 1, p.ny = dx ? 1 : 0, p.ycols = dx ? gu : 0;
  p.split = 192 + gu + d > 512;
  if (dx && (p.split || 192 + gu + p.nc * (gu + d) > 512)) return false;
  const int cols = p.split ? std::max(gu, d) : gu + d;
  p.cpc = std::min(p.nc, (512 - 192 - p.ycols) / cols);
  p.groups = ceil_div(p.nc, p.cpc);
  p.cpc = ceil_div(p.nc, p.groups);
  if (!dx && 2 * 192 + p.cpc * cols <= 512) p.nb = 2;
  p.tmem_cols = pow2_cols(p.nb * 192 + p.ycols + p.cpc * cols);
  if (p.split) p.groups *= 2;
  p.slices = static_cast<int>(std::min<int64_t>(p.tiles, std::max(1, sm_count() / p.groups)));
  p.h_bytes = (p.split ? 2 : 3) * (p.fine ? 2 : 1) * kBlockBytes;
  p.w_bytes = weight_bytes(p, p.cpc);
  int64_t budget = kSmemBudget;
  if (dx) plan_stage(p, p.f.d, 2 * p.tile_bytes + p.h_bytes + p.w_bytes, budget);
  auto used = [&] { return static_cast<int64_t>(p.nx) * p.tile_bytes + p.nh * p.h_bytes; };
  const int tries[][2] = {{3, 2}, {2, 2}, {2, 1}, {1, 2}, {1, 1}};
  p.resident = 1, p.slots = p.slots_f = 0;
  for (const auto& t : tries) {
    p.nx = t[0], p.nh = t[1];
    if (used() + p.w_bytes <= budget) return true;
  }
  if (dx) return false;
  p.resident = 0;
  for (const auto& t : tries) {
    p.nx = t[0], p.nh = t[1];
    p.slots = static_cast<int>(std::min<int64_t>(kMaxSlots, (budget - used()) / kBlockBytes));
    if (p.slots >= 3) break;
  }
  p.slots_f = p.slots;
  return true;
}

uint32_t tc_smem(const TcParams& p) {
  return p.nx * p.tile_bytes + p.nh * p.h_bytes +
         (p.resident ? p.w_bytes : p.slots * kBlockBytes) + p.stage_bytes + 1024;
}

int pack_weights(const TcParams& p, uint8_t* dst, cudaStream_t s) {
  ffn_pack_kernel<<<ceil_div<uint32_t>(weight_bytes(p, p.nc) / 16, 256), 256, 0, s>>>(p, dst);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

template <int kMode, bool kFine = false>
int launch_tc(TcParams p, cudaStream_t s) {
  const int smem = static_cast<int>(tc_smem(p));
  // One limit for calls of every size: it belongs to the kernel, and another
  // thread may be launching it. Before the tensor maps: this binds the thread's
  // context, which a thread of autograd's may not have yet and the encoder needs.
  TGS_CUDA(cudaFuncSetAttribute(ffn_tc_kernel<kMode, kFine>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget + 1024));
  if (int rc = make_maps(p, kMode != kFwd)) return rc;
  const int out = kMode == kFwd ? p.f.o : p.f.d;
  p.vec_y = out % 8 == 0;
  ffn_tc_kernel<kMode, kFine><<<p.groups * p.slices, kTcThreads, smem, s>>>(p);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

// How a backward call runs: as one kernel (`both`), or as one for dX and one
// for the weights' gradients; the laid-out weights follow the partial sums.
struct BwdPlan {
  TcParams rows, weights;
  bool both;
  int64_t partial, floats;
};

BwdPlan plan_backward(const FfnParams& f, bool dx, bool dw) {
  BwdPlan b{};
  b.rows = b.weights = tc_params(f, true);
  b.both = dx && dw && !b.weights.fine && plan_weights(b.weights, true);
  bool packed = false;
  if (dw && !b.both) {
    b.weights = tc_params(f, true);
    plan_weights(b.weights, false);
    packed |= !b.weights.resident;
  }
  if (dx && !b.both) {
    plan_rows(b.rows, true);
    packed |= !b.rows.resident;
  }
  if (dw)
    b.partial = static_cast<int64_t>(b.weights.slices) * b.weights.nc * chunk_floats(b.weights);
  b.floats = b.partial + (packed ? weight_bytes(b.rows, b.rows.nc) / 4 : 0);
  return b;
}

}  // namespace

int make_row_map(CUtensorMap* map, const void* base, int64_t rows, int cols, int64_t stride) {
  static std::atomic<decltype(&cuTensorMapEncodeTiled)> known{nullptr};
  auto encode = known.load(std::memory_order_relaxed);
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    TGS_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found));
    TGS_CHECK_ARG(fn != nullptr, "cuTensorMapEncodeTiled is missing from the driver");
    encode = reinterpret_cast<decltype(encode)>(fn);
    known.store(encode, std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {kBlockCols, 128}, steps[2] = {1, 1};
  const CUresult rc =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box,
             steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d): %lld rows x %d, stride %lld", static_cast<int>(rc),
              static_cast<long long>(rows), cols, static_cast<long long>(stride));
    return TGS_ERR_CUDA;
  }
  return TGS_OK;
}

int ffn_tc_forward(const FfnParams& f, cudaStream_t s) {
  TcParams p = tc_params(f, false);
  plan_rows(p, false);
  if (!p.resident) {
    p.packed = reinterpret_cast<const uint8_t*>(f.scratch);
    if (int rc = pack_weights(p, reinterpret_cast<uint8_t*>(f.scratch), s)) return rc;
  }
  return launch_tc<kFwd, true>(p, s);
}

int64_t ffn_tc_scratch_floats(int64_t n, int d, int h, int o, bool backward) {
  FfnParams f{};
  f.n = n, f.d = d, f.h = h, f.o = o;
  if (!backward) {
    TcParams p = tc_params(f, false);
    plan_rows(p, false);
    return p.resident ? 0 : weight_bytes(p, p.nc) / 4;
  }
  // whichever gradients are asked for
  return std::max(plan_backward(f, true, true).floats,
                  std::max(plan_backward(f, true, false).floats, plan_backward(f, false, true).floats));
}

int ffn_tc_backward(const FfnParams& f, cudaStream_t s) {
  const bool dx = f.y != nullptr, dw = f.dwg != nullptr;
  BwdPlan b = plan_backward(f, dx, dw);
  if (b.floats > b.partial) {
    uint8_t* packed = reinterpret_cast<uint8_t*>(f.scratch + b.partial);
    b.rows.packed = b.weights.packed = packed;
    if (int rc = pack_weights(b.rows, packed, s)) return rc;
  }
  b.weights.partial = f.scratch;
  if (dx && !b.both) {
    if (int rc = b.rows.fine ? launch_tc<kDx, true>(b.rows, s) : launch_tc<kDx>(b.rows, s)) return rc;
  }
  if (!dw) return TGS_OK;
  if (int rc = b.both           ? launch_tc<kDxDw>(b.weights, s)
               : b.weights.fine ? launch_tc<kDw, true>(b.weights, s)
                                : launch_tc<kDw>(b.weights, s))
    return rc;
  ffn_tc_sum_kernel<<<static_cast<unsigned>(b.weights.nc * (chunk_floats(b.weights) / 128)), 256, 0, s>>>(
      b.weights);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

}  // namespace tgs

extern "C" int tgs_align_rows(const void* src, int64_t stride, int64_t n, int32_t c, void* dst,
                              void* stream) {
  using namespace tgs;
  TGS_CHECK_ARG(n >= 0 && c >= 1, "tgs_align_rows: bad sizes (n %lld, c %d)", static_cast<long long>(n),
                c);
  if (n == 0) return TGS_OK;
  TGS_CHECK_ARG(src && dst && aligned16(dst), "tgs_align_rows: NULL or unaligned pointer");
  TGS_CHECK_ARG(n == 1 || stride >= c, "tgs_align_rows: rows overlap (stride %lld, c %d)",
                static_cast<long long>(stride), c);
  const int units = ceil_div(c, 8);
  const int64_t blocks = std::min<int64_t>(ceil_div<int64_t>(n * units, 256), sm_count() * 16ll);
  align_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, as_stream(stream)>>>(
      static_cast<const uint16_t*>(src), stride, n, c, static_cast<uint4*>(dst), units);
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}
