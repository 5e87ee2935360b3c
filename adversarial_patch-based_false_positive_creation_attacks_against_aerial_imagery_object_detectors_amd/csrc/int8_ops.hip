// Matrix product in 8-bit integers with a scale for each token and each output
// channel (po_quantize_rows, po_int8_matmul).
//
//   s[m] = max_k |x[m][k]| / 127      q[m][k] = x[m][k] / s[m] to the nearest, ties to even
//   y[m][n] = (sum_k q[m][k] w[n][k]) * s[m] * sw[n] + bias[n]
//
// The sums are whole numbers in 32 bits (exact: k stays under 2^17); y is
// rounded to its type once.  Weights are the rows (A) of the product and tokens
// its columns, so that a token's outputs are neighbours in a lane.
#include "mm_core.h"
#include <math.h>

namespace {
using namespace po::mm;
using po::ceil_div;

// Elements of the callers' types as fp32.
template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == PO_F32)
    return static_cast<const float*>(p)[i];
  else if constexpr (DT == PO_F16)
    return (float)static_cast<const _Float16*>(p)[i];
  else
    return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

// The quotient x / s rounded to the nearest whole number, ties to even, from the
// exact remainder: x - q s is a multiple of half a step of s and stays within s,
// so the fused multiply-add gives it exactly.
__device__ __forceinline__ int quotient(float x, float s, float inv) {
  float q = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x), half = 0.5f * s;
  const float up = r > 0.f ? 1.f : -1.f;
  if (fabsf(r) > half || (fabsf(r) == half && ((int)q & 1))) q += up;
  return (int)q;
}

// One row to WPR waves.  A row that holds NaN or an infinity gets the scale NaN.
template <int DT, int WPR>
__global__ __launch_bounds__(256) void quantize_rows_k(const void* __restrict__ x, int64_t ldx, int64_t rows, int K,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  constexpr int T = WPR * 64;
  const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + threadIdx.x / T;
  const int t = threadIdx.x % T;
  const int64_t at = row * ldx;
  uint32_t top = 0;
  if (row < rows)
    for (int k = t; k < K; k += T) top = max(top, __float_as_uint(load1<DT>(x, at + k)) & 0x7fffffffu);
  top = po::wave_max_u32(top);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  if (row >= rows) return;
  const bool bad = top >= 0x7f800000u;                       // as bits NaN lies above infinity
  const float s = __uint_as_float(top) / 127.f, inv = 1.f / s;
  if (t == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  const int Kp = (K + 15) / 16 * 16;
  for (int k = t; k < Kp; k += T) {
    int v = 0;
    if (k < K && !bad && s > 0.f) {
      const float f = load1<DT>(x, at + k);
      // 1 / s and half steps of s need normal numbers
      v = s > 1e-30f ? quotient(f, s, inv) : (int)__builtin_rint((double)f / (double)s);
    }
    q[row * ldq + k] = (int8_t)v;
  }
}

template <int DT>
struct ScaledEpi {
  struct Args {
    void* y;
    int64_t ld;
    const float *sx, *sw, *bias;
    int N, M, wide;             // tokens, outputs; wide: rows start on 16 bytes
  };
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, char* lds, const po::mm::Args&) {
    float sx[C::TN];
#pragma unroll
    for (int j = 0; j < C::TN; ++j) sx[j] = t.col(j) < e.N ? e.sx[t.col(j)] : 0.f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = t.row4(i, q);
        float sw[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sw[k] = m + k < e.M ? e.sw[m + k] : 0.f;
          b[k] = e.bias && m + k < e.M ? e.bias[m + k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = __builtin_fmaf((float)t.acc[i][j][4 * q + k] * sx[j], sw[k], b[k]);
          if constexpr (DT == PO_F32) {
            const int n = t.col(j);
            if (n < e.N) {
              float* o = static_cast<float*>(e.y) + (int64_t)n * e.ld + m;
              if (e.wide && m + 4 <= e.M) {
                *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (m + k < e.M) o[k] = v[k];
              }
            }
          } else {
            constexpr int KIND = DT == PO_F16 ? F16 : BF16;
            stage4(t, lds, i, j, q, u2v{pack2<KIND>(v[0], v[1]), pack2<KIND>(v[2], v[3])});
          }
        }
      }
    if constexpr (DT != PO_F32) {
      __syncthreads();
      store_rows<C>(lds, static_cast<uint16_t*>(e.y), e.ld, t.tn * C::BN, t.tm * C::BM, e.N, e.M, e.wide != 0);
    }
  }
};

// Tile by the work: the largest that still gives most CUs one; few tokens: 32 columns.
template <int DT>
int product_of(const Args& a, const typename ScaledEpi<DT>::Args& e, hipStream_t s) {
  using E = ScaledEpi<DT>;
  const char* what = "po_int8_matmul";
  const int64_t M = a.A.rows, N = a.B.rows;
  if (N <= 32) return launch_product<Cfg<I8, 128, 32, 4, 1, 128, 3>, E>(a, e, 1, s, what);
  if ((int64_t)ceil_div(M, 256) * ceil_div(N, 256) >= 192) return launch_product<Cfg<I8, 256, 256, 2, 4, 128, 2>, E>(a, e, 1, s, what);
  if ((int64_t)ceil_div(M, 128) * ceil_div(N, 128) >= 192) return launch_product<Cfg<I8, 128, 128, 2, 2, 128, 2>, E>(a, e, 1, s, what);
  return launch_product<Cfg<I8, 64, 64, 2, 2, 128, 3>, E>(a, e, 1, s, what);
}

inline int element_bytes(int dtype) { return dtype == PO_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == PO_F32 || dtype == PO_F16 || dtype == PO_BF16; }

}  // namespace

extern "C" int po_quantize_rows(const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                                float* scale, po_stream_t stream) {
  PO_REQUIRE(x && q && scale, "po_quantize_rows: null pointer");
  PO_REQUIRE(known(dtype), "po_quantize_rows: unknown dtype %d", dtype);
  PO_REQUIRE(M >= 1 && M <= (1 << 21) && K >= 1 && K < (1 << 17), "po_quantize_rows: bad sizes (M=%lld K=%lld)", (long long)M,
             (long long)K);
  PO_REQUIRE(ldx >= K && ldq >= (K + 15) / 16 * 16 && ldq % 16 == 0 && (uintptr_t)q % 16 == 0,
             "po_quantize_rows: bad strides");
  const hipStream_t s = po::stream_of(stream);
  const bool wave = K <= 1024;                               // a wave covers such a row in a few steps
  const dim3 grid(wave ? ceil_div(M, 4) : (unsigned)M);
#define PO_Q(DT)                                                                                                       \
  if (wave)                                                                                                            \
    hipLaunchKernelGGL((quantize_rows_k<DT, 1>), grid, dim3(256), 0, s, x, ldx, M, (int)K, q, ldq, scale);             \
  else                                                                                                                 \
    hipLaunchKernelGGL((quantize_rows_k<DT, 4>), grid, dim3(256), 0, s, x, ldx, M, (int)K, q, ldq, scale);
  if (dtype == PO_F32) {
    PO_Q(PO_F32)
  } else if (dtype == PO_F16) {
    PO_Q(PO_F16)
  } else {
    PO_Q(PO_BF16)
  }
#undef PO_Q
  return po::check_launch("po_quantize_rows");
}

extern "C" int po_int8_matmul(const int8_t* q, int64_t ldq, const float* sx, const int8_t* w, int64_t ldw,
                              const float* sw, const float* bias, int64_t M, int64_t N, int64_t K, void* y, int64_t ldy,
                              int dtype, po_stream_t stream) {
  PO_REQUIRE(q && sx && w && sw && y, "po_int8_matmul: null pointer");
  PO_REQUIRE(known(dtype), "po_int8_matmul: unknown dtype %d", dtype);
  PO_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= (1 << 21) && N <= (1 << 24) && K < (1 << 17),
             "po_int8_matmul: bad sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  const int64_t Kp = (K + 15) / 16 * 16;
  PO_REQUIRE(ldq >= Kp && ldq % 16 == 0 && (uintptr_t)q % 16 == 0 && ldw >= Kp && ldw % 16 == 0 && (uintptr_t)w % 16 == 0 &&
                 ldq <= (1 << 22) && ldw <= (1 << 22) && ldy >= N,
             "po_int8_matmul: rows must start on 16 bytes and be laid out to a multiple of 16");
  Args a{};
  a.A = Operand{reinterpret_cast<const char*>(w), ldw, 0, (int)N};
  a.B = Operand{reinterpret_cast<const char*>(q), ldq, 0, (int)M};
  a.kbytes = (int)Kp;
  a.pairs = 1;
  const int es = element_bytes(dtype);
  const int wide = (uintptr_t)y % 16 == 0 && ldy * es % 16 == 0;
  const hipStream_t s = po::stream_of(stream);
  if (dtype == PO_F32) return product_of<PO_F32>(a, {y, ldy, sx, sw, bias, (int)M, (int)N, wide}, s);
  if (dtype == PO_F16) return product_of<PO_F16>(a, {y, ldy, sx, sw, bias, (int)M, (int)N, wide}, s);
  return product_of<PO_BF16>(a, {y, ldy, sx, sw, bias, (int)M, (int)N, wide}, s);
}
