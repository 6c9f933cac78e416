// Dropout whose mask is recomputed instead of stored: the decision for
// (row id, column) is a word of a counter-based generator, so the backward
// pass, and any rank or slot that holds the same Gaussian, draws it again.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011). Key = the 64-bit seed, counter =
// (id low, id high, column / 4, offset), word column % 4; a value is kept if
// its word >= floor(p 2^32), and kept values are multiplied by 1 / (1 - p).
// Dropped values become zero by selection, so NaN or infinity there is gone.
//
// Bound: HBM for 32-bit rows of several columns (one generator call serves
// four of them): 1,048,576 rows of 64 fp32 97 us (5.5 TB/s, 86 % of the copy
// rate). 16-bit rows: the generator, whose wide products keep the half of the
// multiply-add units that has them 64 % busy, the logical operations the other
// arithmetic 54 %, with registers for 5.5 warps to a scheduler (the four items
// in flight) between whose loads that work stands: of 64 bf16 82 us (3.3 TB/s).
// Single columns have a generator call each: 4,194,304 rows of one fp32 value
// by ids 27 us. With per_row every item of a row draws its word again: of 64
// fp32 91 us, of 64 bf16 59.
#include "tgs_common.cuh"
#include "tgs_vec.cuh"

namespace tgs {
namespace {

constexpr int kDropThreads = 256;
constexpr int kDropItems = 4;  // items (one load each) in flight per thread
constexpr int kDropMaxC = 65536;

struct DropParams {
  const void* x;
  void* y;
  const int64_t* ids;
  const int64_t* offset_dev;
  int64_t n, x_stride;
  uint64_t limit;  // 2^32 drops everything
  uint32_t key0, key1, offset;
  uint32_t per_row;  // items per row
  uint32_t magic;    // ceil(2^32 / per_row)
  int c, row_wise;
  float scale;
};

__device__ __forceinline__ void philox4x32_10(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c[0];
    const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c[2];
    c[0] = static_cast<uint32_t>(p1 >> 32) ^ c[1] ^ (k0 + r * 0x9E3779B9u);
    c[2] = static_cast<uint32_t>(p0 >> 32) ^ c[3] ^ (k1 + r * 0xBB67AE85u);
    c[1] = static_cast<uint32_t>(p1);
    c[3] = static_cast<uint32_t>(p0);
  }
}

// One item = kVec neighbouring columns of one row; kVec 16-byte loads where
// the rows allow them (kWhole), else four columns one by one.
template <class T, int kVec, bool kWhole>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const DropParams p) {
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const uint32_t step = p.offset_dev ? static_cast<uint32_t>(*p.offset_dev) : p.offset;
  const int64_t items = p.n * p.per_row;
  constexpr int kTile = kDropThreads * kDropItems;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTile; base < items;
       base += static_cast<int64_t>(gridDim.x) * kTile) {
    const int64_t row0 = base / p.per_row;
    const uint32_t rem = static_cast<uint32_t>(base - row0 * p.per_row);
    float v[kDropItems][kVec];
    int64_t row[kDropItems], id[kDropItems];
    uint32_t col[kDropItems];
#pragma unroll
    for (int k = 0; k < kDropItems; ++k) {
      // rem + tile < 2^15 and per_row <= 2^14: the product by magic is exact
      const uint32_t e = rem + k * kDropThreads + threadIdx.x;
      const uint32_t q = p.per_row == 1 ? e : __umulhi(e, p.magic);
      row[k] = row0 + q;
      col[k] = (e - q * p.per_row) * kVec;
      const bool on = row[k] < p.n;
      id[k] = p.ids && on ? p.ids[row[k]] : row[k];
      if constexpr (kWhole) {
        load_vec<T, kVec>(x + row[k] * p.x_stride + col[k], on, v[k]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          v[k][i] = on && col[k] + i < p.c ? to_f32(x[row[k] * p.x_stride + col[k] + i]) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < kDropItems; ++k) {
      if (row[k] >= p.n) continue;
#pragma unroll
      for (int g = 0; g < kVec; g += 4) {
        uint32_t w[4] = {static_cast<uint32_t>(id[k]), static_cast<uint32_t>(id[k] >> 32),
                         p.row_wise ? 0u : (col[k] + g) >> 2, step};
        philox4x32_10(w, p.key0, p.key1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool keep = (p.row_wise ? w[0] : w[i]) >= p.limit;
          v[k][g + i] = keep ? v[k][g + i] * p.scale : 0.f;
        }
      }
      T* dst = y + row[k] * p.c + col[k];
      if constexpr (kWhole) {
        store_vec<T, kVec>(dst, v[k]);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (col[k] + i < p.c) dst[i] = from_f32<T>(v[k][i]);
      }
    }
  }
}

template <class T>
int launch_dropout(DropParams p, cudaStream_t s) {
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = p.c % kWide == 0 && p.x_stride % kWide == 0 && aligned16(p.x) && aligned16(p.y);
  p.per_row = wide ? p.c / kWide : ceil_div(p.c, 4);
  p.magic = static_cast<uint32_t>(((1ull << 32) + p.per_row - 1) / p.per_row);
  const int64_t tiles = ceil_div<int64_t>(p.n * p.per_row, kDropThreads * kDropItems);
  const int grid = static_cast<int>(std::min<int64_t>(tiles, static_cast<int64_t>(sm_count()) * 16));
  if (wide) {
    dropout_kernel<T, kWide, true><<<grid, kDropThreads, 0, s>>>(p);
  } else {
    dropout_kernel<T, 4, false><<<grid, kDropThreads, 0, s>>>(p);
  }
  TGS_LAUNCH_CHECK();
  return TGS_OK;
}

}  // namespace
}  // namespace tgs

using namespace tgs;

extern "C" int tgs_dropout(const TgsDropoutArgs* a, void* stream) {
  TGS_CHECK_ARG(a != nullptr, "tgs_dropout: args is NULL");
  TGS_CHECK_ARG(a->n >= 0 && a->c >= 1 && a->c <= kDropMaxC, "tgs_dropout: bad sizes (n %lld, c %d)",
                static_cast<long long>(a->n), a->c);
  TGS_CHECK_ARG(valid_dtype(a->dtype), "tgs_dropout: unknown type");
  TGS_CHECK_ARG(a->p >= 0.0 && a->p <= 1.0, "tgs_dropout: p %g is not in [0, 1]", a->p);
  if (a->n == 0) return TGS_OK;
  TGS_CHECK_ARG(a->x && a->y, "tgs_dropout: NULL pointer");
  TGS_CHECK_ARG(a->n == 1 || a->x_stride >= a->c, "tgs_dropout: rows overlap (stride %lld, c %d)",
                static_cast<long long>(a->x_stride), a->c);
  DropParams p{};
  p.x = a->x, p.y = a->y, p.ids = a->ids, p.offset_dev = a->offset_dev;
  p.n = a->n, p.x_stride = a->x_stride, p.c = a->c, p.row_wise = a->per_row;
  p.limit = static_cast<uint64_t>(a->p * 4294967296.0);
  p.key0 = static_cast<uint32_t>(a->seed), p.key1 = static_cast<uint32_t>(a->seed >> 32);
  p.offset = a->offset;
  p.scale = a->p < 1.0 ? static_cast<float>(1.0 / (1.0 - a->p)) : 0.f;
  cudaStream_t s = as_stream(stream);
  switch (a->dtype) {
    case TGS_F32: return launch_dropout<float>(p, s);
    case TGS_BF16: return launch_dropout<__nv_bfloat16>(p, s);
    default: return launch_dropout<__half>(p, s);
  }
}
