// Dropout whose mask is a function of a key (po_dropout): never stored, drawn
// again by the backward pass, the same for a row whichever rank holds it.
//
//   y[r][c] = (u >= drop ? x[r][c] * 65536 / (65536 - drop) : 0) [+ residual[r][c]]
//
// u: 16 bits of Philox4x32-10 with key {seed lo, seed hi ^ tag} and counter
// {c / 8, row0 + r, step lo, step hi}: element c of a row takes half c % 2 of
// word (c % 8) / 2.  The tag keeps these numbers apart from po_draws', which have
// the same counters.  16 bits: the keep probability is a multiple of 2^-16, and the
// scale is that probability's, so the mean is x exactly.  32 bits a number would
// double the generator's work (20 products of 32 x 32 bits for each 4 elements),
// which would then bound the kernel instead of the memory.
#pragma clang fp contract(off)
#include "common.h"
#include "philox.h"
#include <algorithm>

namespace {

constexpr uint32_t kTag = 0x64726F70u;

struct F32 {
  using vec = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
struct F16 {
  using vec = _Float16;
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
struct BF16 {
  using vec = __bf16;
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

// One thread: 8 elements of a row (one generator call), wherever the row starts (global
// loads and stores need no alignment; 16 bytes at odd places cost little: 1203 x 1001
// fp32 with residual 9.9 us element by element, 4.6 this way).  A row's last elements go
// one by one.
template <class T, bool RES>
__global__ __launch_bounds__(256) void dropout_k(const typename T::vec* x, int64_t ldx, const typename T::vec* res,
                                                 int64_t ldr, int64_t rows, int64_t cols, uint32_t k0, uint32_t k1,
                                                 uint64_t step, const int64_t* __restrict__ step_dev,
                                                 int64_t* __restrict__ step_used, uint32_t row0, uint32_t drop,
                                                 float scale, typename T::vec* y, int64_t ldy) {
  typedef typename T::vec V;
  typedef V v8 __attribute__((ext_vector_type(8), aligned(sizeof(V))));
  if (step_dev) step = (uint64_t)*step_dev;
  if (step_used && blockIdx.x == 0 && threadIdx.x == 0) *step_used = (int64_t)step;
  const int64_t groups = (cols + 7) / 8, total = rows * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups, g = i - r * groups;
    const V* xp = x + r * ldx + 8 * g;
    const V* rp = RES ? res + r * ldr + 8 * g : nullptr;
    V* yp = y + r * ldy + 8 * g;
    const int m = (int)min((int64_t)8, cols - 8 * g);
    v8 a, b;
    if (m == 8) {
      a = *reinterpret_cast<const v8*>(xp);
      if constexpr (RES) b = *reinterpret_cast<const v8*>(rp);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        a[k] = k < m ? xp[k] : (V)0;
        if constexpr (RES) b[k] = k < m ? rp[k] : (V)0;
      }
    }
    const po::u4 w = po::philox4x32_10(po::u4{(uint32_t)g, row0 + (uint32_t)r, (uint32_t)step, (uint32_t)(step >> 32)}, k0, k1);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    v8 o;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t n = k & 1 ? u[k >> 1] >> 16 : u[k >> 1] & 0xffffu;
      float v = n >= drop ? T::get(a[k]) * scale : 0.f;
      if constexpr (RES) v += T::get(b[k]);
      o[k] = T::put(v);
    }
    if (m == 8) {
      *reinterpret_cast<v8*>(yp) = o;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < m) yp[k] = o[k];
    }
  }
}

template <class T>
int run(const void* x, int64_t ldx, const void* res, int64_t ldr, int64_t rows, int64_t cols, uint64_t seed,
        uint64_t step, const int64_t* step_dev, int64_t* step_used, int64_t row0, int drop, void* y, int64_t ldy,
        hipStream_t s) {
  typedef typename T::vec V;
  const V *xp = static_cast<const V*>(x), *rp = static_cast<const V*>(res);
  V* yp = static_cast<V*>(y);
  const int64_t total = rows * ((cols + 7) / 8);
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((total + 255) / 256, 256 * 32));
  const float scale = drop == 65536 ? 0.f : (float)(65536.0 / (65536 - drop));
#define PO_D(RES)                                                                                                    \
  hipLaunchKernelGGL((dropout_k<T, RES>), dim3(grid), dim3(256), 0, s, xp, ldx, rp, ldr, rows, cols, (uint32_t)seed,   \
                     (uint32_t)(seed >> 32) ^ kTag, step, step_dev, step_used, (uint32_t)row0, (uint32_t)drop, scale, yp, ldy)
  if (res) PO_D(true);
  else PO_D(false);
#undef PO_D
  return po::check_launch("po_dropout");
}

}  // namespace

extern "C" int po_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, int dtype, int64_t rows,
                          int64_t cols, uint64_t seed, uint64_t step, const int64_t* step_dev, int64_t* step_used,
                          int64_t row0, int drop, void* y, int64_t ldy, po_stream_t s) {
  PO_REQUIRE(x && y, "po_dropout: null pointer");
  PO_REQUIRE(drop >= 0 && drop <= 65536, "po_dropout: drop must be in [0, 65536]");
  PO_REQUIRE(rows >= 1 && cols >= 1 && row0 >= 0 && row0 + rows <= (1LL << 32) && cols <= (1LL << 34),
             "po_dropout: bad sizes (rows=%lld cols=%lld row0=%lld)", (long long)rows, (long long)cols, (long long)row0);
  PO_REQUIRE(ldx >= cols && ldy >= cols && (!residual || ldr >= cols), "po_dropout: bad row strides");
  const hipStream_t st = po::stream_of(s);
  switch (dtype) {
    case PO_F32: return run<F32>(x, ldx, residual, ldr, rows, cols, seed, step, step_dev, step_used, row0, drop, y, ldy, st);
    case PO_F16: return run<F16>(x, ldx, residual, ldr, rows, cols, seed, step, step_dev, step_used, row0, drop, y, ldy, st);
    case PO_BF16: return run<BF16>(x, ldx, residual, ldr, rows, cols, seed, step, step_dev, step_used, row0, drop, y, ldy, st);
  }
  PO_REQUIRE(false, "po_dropout: unknown dtype %d", dtype);
}
