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

// n <= 8 neighbouring elements as fp32, wherever they start (global loads need no alignment); 0 past n.
template <int DT>
struct Elem {
  using type = uint16_t;
  static __device__ __forceinline__ float f(uint16_t v) {
    if constexpr (DT == PO_F16)
      return (float)__builtin_bit_cast(_Float16, v);
    else
      return __uint_as_float((uint32_t)v << 16);
  }
};
template <>
struct Elem<PO_F32> {
  using type = float;
  static __device__ __forceinline__ float f(float v) { return v; }
};
template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, int n, float* v) {
  typedef typename Elem<DT>::type T;
  typedef T v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const T* p = static_cast<const T*>(x) + at;
  if (n >= 8) {
    const v8 r = *reinterpret_cast<const v8*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = Elem<DT>::f(r[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? Elem<DT>::f(p[k]) : 0.f;
  }
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

// A row's scale, from the bits of its largest |x|, and the 8-bit numbers under it.
struct RowScale {
  float s, inv;
  bool bad;                                                  // the row holds NaN or an infinity: as bits they lie on top
  __device__ __forceinline__ explicit RowScale(uint32_t top) : s(__uint_as_float(top) / 127.f), inv(1.f / s), bad(top >= 0x7f800000u) {}
  __device__ __forceinline__ float stored() const { return bad ? __uint_as_float(0x7fc00000u) : s; }
  // 8 bits each, of eight
  __device__ __forceinline__ uint2 quotients(const float* v) const {
    uint32_t b[2] = {0, 0};
    if (!bad && s > 1e-30f) {
      // Where every remainder stays below half of s the rounded products are the quotients (ties, and values next to
      // one, are looked at one by one); added to 1.5 * 2^23 their low byte is the number.
      float q[8], far = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[j] = __builtin_rintf(v[j] * inv);
        far = fmaxf(far, fabsf(__builtin_fmaf(-q[j], s, v[j])));
      }
      if (far >= 0.5f * s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = (float)quotient(v[j], s, inv);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(q[4 * h + j] + 12582912.f);
        b[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400), __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400), 0x05040100);
      }
    } else if (!bad && s > 0.f) {
      // 1 / s and half steps of s need normal numbers.  A scale of few bits (below 127 * 2^-149) can lie so far below
      // the largest / 127 that quotients pass 127: those are 127.
#pragma unroll 1
      for (int h = 0; h < 2; ++h)
#pragma unroll 1
        for (int j = 3; j >= 0; --j) {
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x = i == h * 4 + j ? v[i] : x;
          const uint32_t n = (uint32_t)(max(-127, min(127, (int)__builtin_rint((double)x / (double)s))) & 255);
          if (h) b[1] = b[1] << 8 | n;
          else b[0] = b[0] << 8 | n;
        }
    }
    return make_uint2(b[0], b[1]);
  }
};

// One row to WPR waves, 8 elements to a lane and step; rows of up to STEPS steps stay
// in registers between the maximum and the quotients, longer ones (STEPS = 0) are read
// again.  A row that holds NaN or an infinity gets the scale NaN.
template <int DT, int WPR, int STEPS>
__global__ __launch_bounds__(256) void quantize_rows_k(const void* __restrict__ x, int64_t ldx, int64_t rows, int K,
                                                       int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
  __shared__ uint32_t tops[4];
  constexpr int T = WPR * 64;
  const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + threadIdx.x / T;
  const int t = threadIdx.x % T;
  const int64_t at = row * ldx;
  const int mine = row < rows ? K : 0;
  const int Kp = (K + 15) / 16 * 16;
  float v[STEPS ? STEPS : 1][8];
  uint32_t top = 0;
  auto top8 = [&](const float* w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(w[j]) & 0x7fffffffu);
  };
  if constexpr (STEPS > 0) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) load8<DT>(x, at + (i * T + t) * 8, mine - (i * T + t) * 8, v[i]);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) top8(v[i]);
  } else {
    for (int k = t * 8; k < mine; k += T * 8) {
      load8<DT>(x, at + k, mine - k, v[0]);
      top8(v[0]);
    }
  }
  top = po::wave_max_u32(top);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  if (row >= rows) return;
  const RowScale r(top);
  if (t == 0) scale[row] = r.stored();
  auto put8 = [&](int k, const float* w) {
    if (k < Kp) *reinterpret_cast<uint2*>(q + row * ldq + k) = r.quotients(w);
  };
  if constexpr (STEPS > 0) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) put8((i * T + t) * 8, v[i]);
  } else {
    for (int k = t * 8; k < Kp; k += T * 8) {
      load8<DT>(x, at + k, mine - k, v[0]);
      put8(k, v[0]);
    }
  }
}

// ---- few tokens ----------------------------------------------------------
// Up to 32 tokens: the weights' bytes are the work (67 MB of 8192 x 8192: 13 us at
// 5.2 TB/s).  A workgroup owns 16 weight rows, its 16 waves slices of k of 256 bytes: a lane's
// loads of 16 bytes (row lane % 16, 64 bytes of a row to a load) are in flight together, and
// go into the matrix cores as they are.  The waves' sums meet in LDS.  FUSED (up to 4
// tokens): the workgroup quantises the tokens itself, into LDS, behind its weights' loads: one
// launch, where the quantisation alone takes 4 us.  One token of 4096 x 4096 takes 6.2 us,
// 8192 x 8192 15; with 4 waves and four times the loads 1.4 and 2.2 us more; with streaming
// (non-temporal) loads 8192 x 8192 1 us more.
constexpr int kFewWaves = 16, kFewLoads = 4, kFewSlice = kFewLoads * 64;
constexpr int kFewLds = 44 << 10;                            // of the 8-bit tokens; with the sums below 64 KB

// A token's row of 8-bit numbers in LDS and its scale, made by the whole workgroup.  A row of
// up to 8192 stays in registers between the maximum and the quotients.  tops: the waves'
// maxima, of every second token the same (one barrier a token).
template <int DT>
__device__ __forceinline__ void quantize_to_lds(const void* x, int64_t at, int K, int Kp, int8_t* q, uint32_t* tops,
                                                float* scale) {
  constexpr int T = kFewWaves * 64;
  uint32_t top = 0;
  float v[8];
  for (int k = threadIdx.x * 8; k < K; k += T * 8) {
    load8<DT>(x, at + k, K - k, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  top = po::wave_max_u32(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = 0;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) top = max(top, tops[w]);
  const RowScale r(top);
  if (threadIdx.x == 0) *scale = r.stored();
  for (int k = threadIdx.x * 8; k < Kp; k += T * 8) {
    if (K > T * 8 || k >= K) load8<DT>(x, at + k, K - k, v);
    *reinterpret_cast<uint2*>(q + k) = r.quotients(v);
  }
}

template <int DT, int TB, bool FUSED>
__global__ __launch_bounds__(kFewWaves * 64) void few_tokens_k(const void* __restrict__ x, int64_t ldx, const int8_t* __restrict__ q,
                                                    int64_t ldq, const float* __restrict__ sx, const int8_t* __restrict__ w,
                                                    int64_t ldw, const float* __restrict__ sw,
                                                    const float* __restrict__ bias, int M, int N, int K,
                                                    void* __restrict__ y, int64_t ldy) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ i4v sums[kFewWaves][TB][64];
  __shared__ uint32_t tops[2][kFewWaves];
  __shared__ float scales[32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, Kp = (K + 15) / 16 * 16;
  const int row = n0 + (lane & 15), quad = lane >> 4;
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + (int64_t)n0 * ldw), 0,
                                                                     0x7fffffff, 0x00020000);
  const uint32_t wat = row < N ? (uint32_t)((lane & 15) * (int)ldw) : kOOB;
  i4v a[kFewLoads];
  auto weights = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kFewLoads; ++j) {
      const int k = k0 + j * 64 + quad * 16;
      a[j] = __builtin_bit_cast(i4v, __builtin_amdgcn_raw_buffer_load_b128(rw, k < Kp ? wat + (uint32_t)k : kOOB, 0, 0));
    }
  };
  weights(wave * kFewSlice);
  if constexpr (FUSED) {
    __builtin_amdgcn_sched_barrier(0);
    for (int t = 0; t < M; ++t)
      quantize_to_lds<DT>(x, t * ldx, K, Kp, reinterpret_cast<int8_t*>(lds) + t * Kp, tops[t & 1], scales + t);
    __syncthreads();
  } else if (threadIdx.x < 32) {
    scales[threadIdx.x] = threadIdx.x < M ? sx[threadIdx.x] : 0.f;
  }
  i4v acc[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) acc[b] = i4v{0, 0, 0, 0};
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(q), 0, 0x7fffffff, 0x00020000);
  for (int k0 = wave * kFewSlice; k0 < Kp; k0 += kFewWaves * kFewSlice) {
    if (k0 != wave * kFewSlice) weights(k0);
#pragma unroll
    for (int j = 0; j < kFewLoads; ++j) {
      const int k = k0 + j * 64 + quad * 16;
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        const int t = b * 16 + (lane & 15);
        i4v v = {0, 0, 0, 0};
        if constexpr (FUSED) {
          if (t < M && k < Kp) v = *reinterpret_cast<const i4v*>(lds + t * Kp + k);
        } else {
          v = __builtin_bit_cast(i4v, __builtin_amdgcn_raw_buffer_load_b128(
                                          rq, t < M && k < Kp ? (uint32_t)(t * (int)ldq + k) : kOOB, 0, 0));
        }
        acc[b] = mfma<I8>(a[j], v, acc[b]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < TB; ++b) sums[wave][b][lane] = acc[b];
  __syncthreads();
  if (wave < TB) {
    i4v s = sums[0][wave][lane];
#pragma unroll
    for (int u = 1; u < kFewWaves; ++u) s += sums[u][wave][lane];
    const int t = wave * 16 + (lane & 15), n = n0 + quad * 4;
    if (t < M) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < N) {
          const float v = __builtin_fmaf((float)s[k] * scales[t], sw[n + k], bias ? bias[n + k] : 0.f);
          if constexpr (DT == PO_F32)
            static_cast<float*>(y)[(int64_t)t * ldy + n + k] = v;
          else
            static_cast<uint16_t*>(y)[(int64_t)t * ldy + n + k] = (uint16_t)pack2<DT == PO_F16 ? F16 : BF16>(v, 0.f);
        }
    }
  }
}

template <int DT>
struct ScaledEpi {
  struct Args {
    void* y;
    int64_t ld;
    const float *sx, *sw, *bias;
    int N, M;                   // tokens, outputs
  };
  template <class C>
  struct Pre {
    float sx[C::TN];
    __device__ __forceinline__ void load(const Tile<C>& t, const Args& e) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) sx[j] = t.col(j) < e.N ? e.sx[t.col(j)] : 0.f;
    }
  };
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>& pre, char* lds) {
    float swv[C::TM][4], bv[C::TM][4];
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        swv[i][k] = t.row(i) + k < e.M ? e.sw[t.row(i) + k] : 0.f;
        bv[i][k] = e.bias && t.row(i) + k < e.M ? e.bias[t.row(i) + k] : 0.f;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const int m = t.row(i);
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __builtin_fmaf((float)t.acc[i][j][k] * pre.sx[j], swv[i][k], bv[i][k]);
        if constexpr (DT == PO_F32) {
          const int n = t.col(j);
          if (n < e.N) {
            float* o = static_cast<float*>(e.y) + (int64_t)n * e.ld + m;
            if (m + 4 <= e.M) {
              *reinterpret_cast<f4u*>(o) = f4u{v[0], v[1], v[2], v[3]};
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (m + k < e.M) o[k] = v[k];
            }
          }
        } else {
          constexpr int KIND = DT == PO_F16 ? F16 : BF16;
          stage4(t, lds, i, j, u2v{pack2<KIND>(v[0], v[1]), pack2<KIND>(v[2], v[3])});
        }
      }
    }
    if constexpr (DT != PO_F32) {
      __syncthreads();
      store_rows<C>(lds, static_cast<uint16_t*>(e.y), e.ld, t.tn * C::BN, t.tm * C::BM, e.N, e.M);
    }
  }
};

template <int DT>
int product_of(const Args& a, const typename ScaledEpi<DT>::Args& e, hipStream_t s) {
  using E = ScaledEpi<DT>;
  const char* what = "po_int8_matmul";
  const Plan p = plan_product(a.A.rows, a.B.rows, ceil_div(a.kbytes, 128), Ends{6, 10, false});
  if (p.tile == LARGE) return launch_product<Cfg<I8, 256, 256, 2, 4, 128, 2>, E>(a, e, 1, s, what);
  // 64 x 64 where tiles of 128 x 128 leave CUs without one; where even these do, two groups of waves
  // take the steps in turn (200 x 2000 x 1500 9.7 -> 8.4 us).  64 x 96 where that makes one round of
  // more (1111 x 4001 x 1000, 288 tiles or 192: 15.9 -> 14.3 us)
  if ((int64_t)ceil_div(a.A.rows, 128) * ceil_div(a.B.rows, 128) < 256) {
    const int64_t tm = ceil_div(a.A.rows, 64);
    if (tm * ceil_div(a.B.rows, 64) <= 256) return launch_product<Cfg<I8, 64, 64, 2, 2, 128, 3, 2>, E>(a, e, 1, s, what);
    if (tm * ceil_div(a.B.rows, 96) <= 256) return launch_product<Cfg<I8, 64, 96, 2, 2, 128, 3, 2>, E>(a, e, 1, s, what);
    return launch_product<Cfg<I8, 64, 64, 2, 2, 256, 2>, E>(a, e, 1, s, what);
  }
  return launch_product<Cfg<I8, 128, 128, 2, 2, 128, 2>, E>(a, e, 1, s, what);
}

constexpr int kFewTokens = 32;

// Tokens that a workgroup of few_tokens_k quantises itself.
inline bool fuses(int64_t M, int64_t K) { return M <= 4 && M * ((K + 15) / 16 * 16) <= kFewLds; }

template <int DT>
int few_tokens(bool fused, const void* x, int64_t ldx, const int8_t* q, int64_t ldq, const float* sx, const int8_t* w,
               int64_t ldw, const float* sw, const float* bias, int M, int N, int K, void* y, int64_t ldy, hipStream_t s) {
  const dim3 grid(ceil_div(N, 16));
  if (fused)
    hipLaunchKernelGGL((few_tokens_k<DT, 1, true>), grid, dim3(kFewWaves * 64), M * ((K + 15) / 16 * 16), s, x, ldx, q, ldq, sx, w, ldw,
                       sw, bias, M, N, K, y, ldy);
  else if (M <= 16)
    hipLaunchKernelGGL((few_tokens_k<DT, 1, false>), grid, dim3(kFewWaves * 64), 0, s, x, ldx, q, ldq, sx, w, ldw, sw, bias, M, N, K, y,
                       ldy);
  else
    hipLaunchKernelGGL((few_tokens_k<DT, 2, false>), grid, dim3(kFewWaves * 64), 0, s, x, ldx, q, ldq, sx, w, ldw, sw, bias, M, N, K, y,
                       ldy);
  return po::check_launch("po_int8_matmul");
}

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
  // a wave to a row of up to 2048, a workgroup (of 4) to a longer one
#define PO_Q(DT, WPR, STEPS)                                                                                           \
  hipLaunchKernelGGL((quantize_rows_k<DT, WPR, STEPS>), dim3(ceil_div(M, 4 / WPR)), dim3(256), 0, s, x, ldx, M, (int)K, q, \
                     ldq, scale)
#define PO_QT(DT)                          \
  do {                                     \
    if (K <= 512) PO_Q(DT, 1, 1);          \
    else if (K <= 2048) PO_Q(DT, 1, 4);    \
    else if (K <= 4096) PO_Q(DT, 4, 2);    \
    else if (K <= 8192) PO_Q(DT, 4, 4);    \
    else PO_Q(DT, 4, 0);                   \
  } while (0)
  if (dtype == PO_F32) PO_QT(PO_F32);
  else if (dtype == PO_F16) PO_QT(PO_F16);
  else PO_QT(PO_BF16);
#undef PO_QT
#undef PO_Q
  return po::check_launch("po_quantize_rows");
}

namespace {

int check_matmul(const char* what, const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, int64_t M, int64_t N, int64_t K,
                 int64_t ldy, int dtype) {
  PO_REQUIRE(known(dtype), "%s: unknown dtype %d", what, dtype);
  PO_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= (1 << 21) && N <= (1 << 24) && K < (1 << 17),
             "%s: bad sizes (M=%lld N=%lld K=%lld)", what, (long long)M, (long long)N, (long long)K);
  const int64_t Kp = (K + 15) / 16 * 16;
  PO_REQUIRE(ldq >= Kp && ldq % 16 == 0 && (uintptr_t)q % 16 == 0 && ldw >= Kp && ldw % 16 == 0 && (uintptr_t)w % 16 == 0 &&
                 ldq <= (1 << 22) && ldw <= (1 << 22) && ldy >= N,
             "%s: rows must start on 16 bytes and be laid out to a multiple of 16", what);
  return PO_OK;
}

int matmul(const int8_t* q, int64_t ldq, const float* sx, const int8_t* w, int64_t ldw, const float* sw, const float* bias,
           int64_t M, int64_t N, int64_t K, void* y, int64_t ldy, int dtype, hipStream_t s) {
  if (M <= kFewTokens) {
#define PO_FEW(DT) few_tokens<DT>(false, nullptr, 0, q, ldq, sx, w, ldw, sw, bias, (int)M, (int)N, (int)K, y, ldy, s)
    return dtype == PO_F32 ? PO_FEW(PO_F32) : dtype == PO_F16 ? PO_FEW(PO_F16) : PO_FEW(PO_BF16);
#undef PO_FEW
  }
  Args a{};
  a.A = Operand{reinterpret_cast<const char*>(w), ldw, 0, (int)N};
  a.B = Operand{reinterpret_cast<const char*>(q), ldq, 0, (int)M};
  a.kbytes = (int)((K + 15) / 16 * 16);
  if (dtype == PO_F32) return product_of<PO_F32>(a, {y, ldy, sx, sw, bias, (int)M, (int)N}, s);
  if (dtype == PO_F16) return product_of<PO_F16>(a, {y, ldy, sx, sw, bias, (int)M, (int)N}, s);
  return product_of<PO_BF16>(a, {y, ldy, sx, sw, bias, (int)M, (int)N}, s);
}

// Workspace of po_int8_linear: the tokens' 8-bit rows, then their scales.  Rows a power of two
// apart fall on few memory channels.  Few tokens: an odd number of 64 bytes (17 x 4096 x 8192
// 15.8 -> 14.0 us); tiles load 128 bytes of a row at a time: a multiple of 128, and not of
// 256 (8192^3 507 -> 497 us).
inline int64_t linear_ldq(int64_t M, int64_t K) {
  if (M <= kFewTokens) return ((K + 63) / 64 | 1) * 64;
  const int64_t p = (K + 127) / 128 * 128;
  return p >= 1024 && p % 256 == 0 ? p + 128 : p;
}
inline int64_t linear_bytes(int64_t M, int64_t K) { return M * (K + 260); }

}  // namespace

extern "C" int po_int8_matmul(const int8_t* q, int64_t ldq, const float* sx, const int8_t* w, int64_t ldw,
                              const float* sw, const float* bias, int64_t M, int64_t N, int64_t K, void* y, int64_t ldy,
                              int dtype, po_stream_t stream) {
  PO_REQUIRE(q && sx && w && sw && y, "po_int8_matmul: null pointer");
  const int rc = check_matmul("po_int8_matmul", q, ldq, w, ldw, M, N, K, ldy, dtype);
  if (rc != PO_OK) return rc;
  return matmul(q, ldq, sx, w, ldw, sw, bias, M, N, K, y, ldy, dtype, po::stream_of(stream));
}

extern "C" int po_int8_linear(const void* x, int64_t ldx, const int8_t* w, int64_t ldw, const float* sw, const float* bias,
                              int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* y,
                              int64_t ldy, int dtype, po_stream_t stream) {
  PO_REQUIRE(x && w && sw && y && workspace, "po_int8_linear: null pointer");
  const int64_t ldq = linear_ldq(M, K);
  const int rc = check_matmul("po_int8_linear", static_cast<int8_t*>(workspace), ldq, w, ldw, M, N, K, ldy, dtype);
  if (rc != PO_OK) return rc;
  PO_REQUIRE(ldx >= K, "po_int8_linear: bad strides");
  PO_REQUIRE(workspace_bytes >= linear_bytes(M, K), "po_int8_linear: workspace of %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)linear_bytes(M, K));
  int8_t* q = static_cast<int8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(q + M * ldq);
  if (fuses(M, K)) {
#define PO_FEW(DT) few_tokens<DT>(true, x, ldx, nullptr, 0, nullptr, w, ldw, sw, bias, (int)M, (int)N, (int)K, y, ldy, po::stream_of(stream))
    return dtype == PO_F32 ? PO_FEW(PO_F32) : dtype == PO_F16 ? PO_FEW(PO_F16) : PO_FEW(PO_BF16);
#undef PO_FEW
  }
  const int rq = po_quantize_rows(x, ldx, dtype, M, K, q, ldq, sx, stream);
  if (rq != PO_OK) return rq;
  return matmul(q, ldq, sx, w, ldw, sw, bias, M, N, K, y, ldy, dtype, po::stream_of(stream));
}
