// Softmax cross entropy of a linear head over a large vocabulary, without its
// logits in memory (po_linear_ce_fwd / _bwd, po_linear_ce_frozen_fwd / _bwd).
//
//   l[n][v] = c * h[n] . w[v]        loss[n] = log sum_v exp l[n][v] - l[n][t_n]
//   dl[n][v] = g_n (exp(l[n][v]) / sum_n - [v = t_n])
//   dh = c * dl w                    dw = c * dl^T h
//
// Forward: one product over all of the vocabulary whose epilogue keeps, for
// each tile of vocabulary rows, the maximum and the sum of the exponentials
// of a token (in 32 bits), and the target's logit.  A tile has the vocabulary as
// its rows, so a token's values lie in four lanes, and the reduction stays in
// registers but for two exchanges.  Backward: for one piece of the
// vocabulary after the other, the logits again, dl in their place (16 bits, as
// [n][v] and as [v][n]), then dh += dl w and the piece's rows of dw.  Every
// product has k contiguous in both operands: w and h are transposed for that.
//
// Against a frozen vocabulary dh alone is wanted, and the forward pass can have it: dh_n = c (sum_v
// exp(l) w - ...) / sum_n needs the exponentials up to a factor of the row.  So a piece's are
// stored in 16 bits, as multiples of powers of two, and multiplied with its rows at once
// (KeepEpi, RefSlabEpi); what is left to the backward pass is a scaling.  Two products instead of
// three: bf16 4096 x 32768 x 1024 784 -> 570 us, 8192 x 100000 x 2048 8.2 -> 5.7 ms,
// fp32 4096 x 32768 x 1024 3.84 -> 2.80.  With dw this gains nothing: dw's terms need
// the rows' whole sums first.
//
// Types.  16-bit inputs: exact products, sums in 32 bits; dl is rounded to the
// inputs' type once, as an operand of the matrix cores: half a step against
// each of a row's terms, below the rounding of the gradients themselves, but seen beside it: the
// norm of bf16 gradients is off by 2.0e-3 where 32-bit dl would give 1.7e-3 (8192 x 131072 x 2048), since the target's
// term is most of a gradient.  dl in two planes would cost those products twice their time.  Against a
// frozen vocabulary the target's term is made in 32 bits (1.7e-3), and of up to 8 tokens all of dl.  fp16 has
// too little range for exp(l)/sum: its dl are kept relative to the largest |g_n|,
// times 2^14 (at most 2^14, and normal down to 2^-28).  fp32 inputs: each number
// is the sum of three bf16 (8 + 8 + 8 bits, nearest), and the six leading of the
// nine products are summed in 32 bits; what is left out is below 2^-24 of a
// product.  That is six bf16 products (220 TFLOP/s of fp32 in the loop) where the
// fp32 matrix instructions end at 157.  Of up to 192 tokens, where reading the vocabulary
// counts for more, those instructions take the numbers as they are.
#include "mm_core.h"
#include <math.h>

namespace {
using namespace po::mm;
using po::ceil_div;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kF16Lift = 16384.f;

// plan_product's tiles, of one plane (P = 1) and of three
template <int KIND, int P>
using Large = std::conditional_t<P == 3, Cfg<KIND, 256, 128, 4, 2, 64, 2, 1, 3>, Cfg<KIND, 256, 256, 2, 4, 128, 2>>;
template <int KIND, int P>
using Mid = std::conditional_t<P == 3, Cfg<KIND, 128, 64, 2, 2, 64, 2, 1, 3>,
                               std::conditional_t<KIND == F32, Cfg<KIND, 128, 64, 4, 1, 128, 2>, Cfg<KIND, 128, 128, 2, 2, 128, 2>>>;
template <int KIND, int P>
using Few = std::conditional_t<P == 3, Cfg<KIND, 128, 32, 4, 1, 64, 2, 1, 3>, Cfg<KIND, 128, 32, 4, 1, 128, 3>>;
// of three only
template <int KIND>
using Square = Cfg<KIND, 128, 128, 4, 2, 64, 2, 1, 3>;
template <int KIND>
using Tall = Cfg<KIND, 192, 128, 4, 2, 64, 2, 1, 3>;

// over the four lanes that hold a column
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The rows' upstream gradients.  Of a sum or a mean there is one, and what the rows need of it
// is made where it is used; of single losses (each) grad_rows_k makes ratio and factor.
struct GradOf {
  const float *grad, *count;
  const int64_t* target;
  int64_t ignore, V;
  int each, mean;
  float lift, c;
  const float *ratio, *factor;
  // g_n over the largest |g|, times the lift of fp16; 0: the row takes no part; NaN: its target is none
  __device__ __forceinline__ float of_row(int n) const {
    if (each) return ratio[n];
    const int64_t t = target[n];
    const float g = *grad;
    return t == ignore || g == 0.f ? 0.f : t < 0 || t >= V || g != g ? __uint_as_float(0x7fc00000u) : copysignf(lift, g);
  }
  __device__ __forceinline__ bool live(int n) const { return each ? ratio[n] != 0.f : target[n] != ignore && *grad != 0.f; }
  // what the products' sums are multiplied with in the end
  __device__ __forceinline__ float end() const {
    return each ? *factor : fabsf(*grad) / (mean ? fmaxf(*count, 1.f) : 1.f) / lift * c;
  }
};

// ---- epilogues -----------------------------------------------------------

// partial[tile][n] = {max of l * log2e, sum of 2^(l * log2e - max)} over the tile's vocabulary rows
struct StatsEpi {
  static constexpr Ends kEnds{3, 5.5, false};                // us, see plan_product
  struct Args {
    float2* partial;
    uint32_t* arrived;          // of row_stats_k, which follows: set to 0
    float* tlogit;              // l / c of the target
    const int64_t* target;
    int64_t v0;                 // vocabulary row of A's first
    int tile0;                  // first tile of this launch in partial
    int N, V;                   // tokens, vocabulary rows of this launch
    float k;                    // c * log2e > 0
  };
  template <class C>
  struct Pre {
    int at[C::TN];              // the target's row within this wave's, or none of them
    __device__ __forceinline__ void load(const Tile<C>& t, const Args& e) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const int64_t r = (t.col(j) < e.N ? e.target[t.col(j)] : -1) - e.v0 - t.m0;
        at[j] = r >= 0 && r < C::TM * 16 ? (int)r : -1;
      }
    }
  };
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>& pre, char* lds) {
    float2* mine = reinterpret_cast<float2*>(lds);          // [WM][BN]
    const int quad = t.lane >> 4;
    if (blockIdx.x == 0 && threadIdx.x == 0) *e.arrived = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const bool has = pre.at[j] >= 0 && ((pre.at[j] >> 2) & 3) == quad;
      if (__any(has)) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pre.at[j] == i * 16 + 4 * quad + k) x = t.acc[i][j][k];
        if (has) e.tlogit[t.col(j)] = x;
      }
    }
    if (t.m0 + C::TM * 16 > e.V) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t.row(i) + k >= e.V) {
#pragma unroll
            for (int j = 0; j < C::TN; ++j) t.acc[i][j][k] = -INFINITY;
          }
    }
    // all columns' maxima, then all their sums: the exchanges between lanes overlap
    float mx[C::TN], top[C::TN], s[C::TN];
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      mx[j] = -INFINITY;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[j] = fmaxf(mx[j], t.acc[i][j][k]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) mx[j] = column_max(mx[j]);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      top[j] = mx[j] == -INFINITY ? 0.f : mx[j] * e.k;       // nothing but -inf: no exponent of inf - inf
      s[j] = 0.f;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[j] += __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][k], e.k, -top[j]));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) s[j] = column_sum(s[j]);
    if (t.lane < 16) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
        mine[t.wm * C::BN + t.wn * C::TN * 16 + j * 16 + t.lane] = make_float2(mx[j] == -INFINITY ? -INFINITY : top[j], s[j]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < C::BN; x += C::NW * 64) {
      float2 r = mine[x];
#pragma unroll
      for (int w = 1; w < C::WM; ++w) {
        const float2 o = mine[w * C::BN + x];
        const float m = fmaxf(r.x, o.x), ref = m == -INFINITY ? 0.f : m;
        r = make_float2(m, r.y * __builtin_amdgcn_exp2f(r.x - ref) + o.y * __builtin_amdgcn_exp2f(o.x - ref));
      }
      const int n = t.tn * C::BN + x;
      if (n < e.N) e.partial[(int64_t)(e.tile0 + t.tm) * e.N + n] = r;
    }
  }
};

// dl of a piece of the vocabulary, as [n][v] and as [v][n]; PLANES = 3: as the three bf16 of each number
template <int KIND, int PLANES>
struct DlogitsEpi {
  static constexpr Ends kEnds{6. * PLANES, PLANES > 1 ? 36. : 15., false};
  struct Args {
    const float2* stat;         // {max * log2e, 1 / sum} of a token
    GradOf g;
    int64_t v0;
    int N, Np, V, Vp;           // tokens and vocabulary rows of the piece, and both as laid out
    float k;
    uint16_t *dl, *dlt;         // [N][ldl], [V][ldt]; planes behind each other
    int64_t ldl, ldt, pl, pt;
  };
  template <class C>
  struct Pre {
    float2 stat[C::TN];
    float ratio[C::TN];
    int at[C::TN];
    __device__ __forceinline__ void load(const Tile<C>& t, const Args& e) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const int n = t.col(j);
        const bool in = n < e.N;
        stat[j] = in ? e.stat[n] : make_float2(0.f, 0.f);
        ratio[j] = in ? e.g.of_row(n) : 0.f;
        const int64_t r = (in ? e.g.target[n] : -1) - e.v0 - t.m0;
        at[j] = r >= 0 && r < C::TM * 16 ? (int)r : -1;
      }
    }
  };
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>& pre, char* lds) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);                     // a column block at a time: the accumulators fill the registers
      const float2 st = pre.stat[j];
      const float r = pre.ratio[j], ir = st.y * r;
      const bool live = r != 0.f;                            // rows that take no part may hold anything, NaN too
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][k], e.k, -st.x)) * ir;
          t.acc[i][j][k] = live ? v : 0.f;
        }
      if (__any(pre.at[j] >= 0)) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pre.at[j] == i * 16 + 4 * (t.lane >> 4) + k) t.acc[i][j][k] -= r;
      }
    }
    if (t.m0 + C::TM * 16 > e.V) {                           // vocabulary rows past the end
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t.row(i) + k >= e.V) {
#pragma unroll
            for (int j = 0; j < C::TN; ++j) t.acc[i][j][k] = 0.f;
          }
    }
    if constexpr (KIND == F32) {                             // as it is: small beside the vocabulary
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const int n = t.col(j);
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          const int m = t.row(i);
          if (e.dl && n < e.N && m < e.Vp) *reinterpret_cast<f4v*>(reinterpret_cast<float*>(e.dl) + n * e.ldl + m) = t.acc[i][j];
          if (e.dlt && n < e.Np) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (m + k < e.V) reinterpret_cast<float*>(e.dlt)[(m + k) * e.ldt + n] = t.acc[i][j][k];
          }
        }
      }
    } else {
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      __syncthreads();                                       // the loop's (or the last plane's) reads are over
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          u2v w;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x = t.acc[i][j][2 * k], y = t.acc[i][j][2 * k + 1];
            w[k] = pack2<KIND>(x, y);
            if constexpr (PLANES > 1) {                      // what this plane leaves to the next
              t.acc[i][j][2 * k] = x - __uint_as_float(w[k] << 16);
              t.acc[i][j][2 * k + 1] = y - __uint_as_float(w[k] & 0xffff0000u);
            }
          }
          stage4(t, lds, i, j, w);
        }
      }
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      const int n0 = t.tn * C::BN, m0 = t.tm * C::BM;
      if (e.dl) store_rows<C>(lds, e.dl + p * e.pl, e.ldl, n0, m0, e.N, e.Vp);
      __builtin_amdgcn_sched_barrier(0);
      if (e.dlt) store_columns<C>(lds, e.dlt + p * e.pt, e.ldt, n0, m0, e.Np, e.V);
      __builtin_amdgcn_sched_barrier(0);
    }
    }
  }
};

// The forward pass of a frozen vocabulary: StatsEpi's statistics, and the exponentials themselves, of
// a piece, as [n][v]: exp(l) = 2^r E, E <= 1.  r is the tile's largest l * log2e of a token, rounded up; bf16
// has the range for one r in most tiles, base, with which the next product is an ordinary one
// (4096 x 32768 x 1024: 221 us, 272 with every tile's own): 2^40 over the target's exponential, which
// is one of the row's, so that what E loses below 2^-126 is below 2^-86 of the row's sum.
// fp16: 2^15 E, normal from 2^-29 on.  The target's E is left out: its part of
// the gradient, p_t - 1, is made in 32 bits.  refs[v / 128][n] = r (-infinity where all E are 0); other[v / 128][n / 32]: there is
// one beside base among those.
template <int KIND, int PLANES>
struct KeepEpi {
  static constexpr Ends kEnds{6. * PLANES, PLANES > 1 ? 30. : 15., false};
  static constexpr float kLift = KIND == F16 ? 15.f : 0.f;
  // a tile's r, from its largest l * log2e; base: frozen_base_k's
  static __device__ __forceinline__ float reference(float top, float base) {
    return base == INFINITY ? 0.f : top <= base ? base : __builtin_ceilf(top);
  }
  struct Args {
    StatsEpi::Args s;
    const float* base;          // frozen_base_k's of the tokens; null: a tile's own r
    float* refs;                // of this launch's first 128 vocabulary rows
    uint8_t* other;
    int64_t ldr, ldo;
    int Vp;                     // vocabulary rows of the launch as laid out
    uint16_t* kept;             // [N][ld]; planes behind each other
    int64_t ld, plane;
  };
  template <class C>
  using Pre = NoPre;
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& a, const NoPre&, char* lds) {
    float(*const mine)[C::BN] = reinterpret_cast<float(*)[C::BN]>(lds);                // [WM]: maxima, then [WM]: sums
    const StatsEpi::Args& e = a.s;
    typename StatsEpi::Pre<C> pre;                           // read here: LARGE has no registers for it in the loop
    pre.load(t, e);
    float base[C::TN];
#pragma unroll
    for (int j = 0; j < C::TN; ++j) base[j] = a.base && t.col(j) < e.N ? a.base[t.col(j)] : __uint_as_float(0x7fc00000u);
    if (blockIdx.x == 0 && threadIdx.x == 0) *e.arrived = 0;
    if (t.m0 + C::TM * 16 > e.V) {
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t.row(i) + k >= e.V) {
#pragma unroll
            for (int j = 0; j < C::TN; ++j) t.acc[i][j][k] = -INFINITY;
          }
    }
    float mx[C::TN];
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      mx[j] = -INFINITY;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[j] = fmaxf(mx[j], t.acc[i][j][k]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) mx[j] = column_max(mx[j]);
    __syncthreads();                                         // the loop's reads are over
    const int c0 = t.wn * C::TN * 16 + (t.lane & 15);
    if (t.lane < 16) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) mine[t.wm][c0 + j * 16] = mx[j];
    }
    __syncthreads();
    float s[C::TN];
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      float top = mine[0][c0 + j * 16];
#pragma unroll
      for (int w = 1; w < C::WM; ++w) top = fmaxf(top, mine[w][c0 + j * 16]);
      top = reference(top * e.k, base[j]);
      const bool none = base[j] == INFINITY;  // the row takes no part
      const float ref = (top == -INFINITY ? 0.f : top) - kLift;
      const bool has = pre.at[j] >= 0 && ((pre.at[j] >> 2) & 3) == t.lane >> 4;
      if (__any(has)) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pre.at[j] == i * 16 + 4 * (t.lane >> 4) + k) x = t.acc[i][j][k];
        if (has) e.tlogit[t.col(j)] = x;
      }
      s[j] = 0.f;
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][k], e.k, -ref));
          t.acc[i][j][k] = none ? 0.f : x;
          s[j] += t.acc[i][j][k];
        }
      if (__any(has)) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (pre.at[j] == i * 16 + 4 * (t.lane >> 4) + k) t.acc[i][j][k] = 0.f;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) s[j] = column_sum(s[j]);
    if (t.lane < 16) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) mine[C::WM + t.wm][c0 + j * 16] = s[j];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < C::BN; x += C::NW * 64) {
      float top = mine[0][x], sum = mine[C::WM][x];
#pragma unroll
      for (int w = 1; w < C::WM; ++w) {
        top = fmaxf(top, mine[w][x]);
        sum += mine[C::WM + w][x];
      }
      const int n = t.tn * C::BN + x;
      bool is_other = false;
      if (n < e.N) {
        const float base = a.base ? a.base[n] : __uint_as_float(0x7fc00000u);
        top = reference(top * e.k, base);
        is_other = top != base && base != INFINITY;
        e.partial[(int64_t)(e.tile0 + t.tm) * e.N + n] = make_float2(top, sum * (kLift ? 0x1p-15f : 1.f));
        // an infinite maximum: E is NaN, and the sums with it, whatever they are multiples of
#pragma unroll
        for (int b = 0; b < C::BM / 128; ++b)
          a.refs[(int64_t)(t.tm * (C::BM / 128) + b) * a.ldr + n] = top == INFINITY ? 0.f : top;
      }
      const uint64_t others = __ballot(is_other);
      if (t.lane % 32 == 0 && n < e.N) {
#pragma unroll
        for (int b = 0; b < C::BM / 128; ++b)
          a.other[(int64_t)(t.tm * (C::BM / 128) + b) * a.ldo + n / 32] = (uint8_t)((uint32_t)(others >> t.lane) != 0);
      }
    }
#pragma unroll
    for (int q = 0; q < PLANES; ++q) {
      __syncthreads();                                       // the loop's (or the last plane's) reads are over
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          u2v w;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x = t.acc[i][j][2 * k], y = t.acc[i][j][2 * k + 1];
            w[k] = pack2<KIND>(x, y);
            if constexpr (PLANES > 1) {                      // what this plane leaves to the next
              t.acc[i][j][2 * k] = x - __uint_as_float(w[k] << 16);
              t.acc[i][j][2 * k + 1] = y - __uint_as_float(w[k] & 0xffff0000u);
            }
          }
          stage4(t, lds, i, j, w);
        }
      }
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      store_rows<C>(lds, a.kept + q * a.plane, a.ld, t.tn * C::BN, t.tm * C::BM, e.N, a.Vp);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The sums of a product with references: slab[slice][n][m] (+)= acc, with the power of two of a slice's
// row in out_refs[slice][n] (in_refs: of what the slab holds).
struct RefSlabEpi {
  static constexpr Ends kEnds{8, 12, true};
  static constexpr bool kRefs = true;
  struct Args {
    const float *refs, *base;   // [k / 128][ldr], [N]
    const uint8_t* other;       // [k / 128][ldo]
    int64_t ldr, ldo;
    int blocks;
    float* slab;
    int64_t ld, slice;          // ld a multiple of 4
    int N, M;
    const float* in_refs;       // [slices][ldr], null: the slab holds nothing
    float* out_refs;
  };
  template <class C>
  using Pre = NoPre;
  template <class C>
  static __device__ __forceinline__ bool plain(const Tile<C>& t, const Args& e) {
    constexpr int PER = C::BN / 32;
    const int first = t.tn * PER, here = min(PER, (int)e.ldo - first);
    int other = 0;
    for (int i = threadIdx.x; i < e.blocks * PER; i += C::NW * 64)
      if (i % PER < here) other |= e.other[(int64_t)(i / PER) * e.ldo + first + i % PER];
    return !__syncthreads_or(other);
  }
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>&, const float (&last)[C::TN]) {
    float* out = e.slab + blockIdx.y * e.slice;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);                     // a column block at a time: the accumulators fill the registers
      const int n = t.col(j);
      if (n >= e.N) continue;
      const float mine = last[j], held = e.in_refs ? e.in_refs[blockIdx.y * e.ldr + n] : -INFINITY;
      const float r = fmaxf(mine, held);
      // sums of nothing but zeros have no power of two
      const float fm = mine == -INFINITY ? 0.f : Refs<C>::pow2(mine - r), fh = held == -INFINITY ? 0.f : Refs<C>::pow2(held - r);
      if (t.tm == 0 && t.wm == 0 && t.lane < 16) e.out_refs[blockIdx.y * e.ldr + n] = r;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int m = t.row(i);
        if (m >= e.ld) continue;
        f4v* o = reinterpret_cast<f4v*>(out + (int64_t)n * e.ld + m);
        *o = e.in_refs ? *o * fh + t.acc[i][j] * fm : t.acc[i][j];
      }
    }
  }
};

// slab[slice][n][m] (+)= acc in 32 bits: the sums of dh over slices of a piece's k and over the pieces
struct SlabEpi {
  static constexpr Ends kEnds{8, 12, true};
  struct Args {
    float* slab;
    int64_t ld, slice;          // ld a multiple of 4
    int N, M, add;
  };
  template <class C>
  using Pre = NoPre;
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>&, char*) {
    float* out = e.slab + blockIdx.y * e.slice;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      __builtin_amdgcn_sched_barrier(0);                     // a column block at a time: the accumulators fill the registers
      const int n = t.col(j);
      if (n >= e.N) continue;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) {
        const int m = t.row(i);
        if (m >= e.ld) continue;
        f4v* o = reinterpret_cast<f4v*>(out + (int64_t)n * e.ld + m);
        *o = e.add ? *o + t.acc[i][j] : t.acc[i][j];
      }
    }
  }
};

// out[n][m] = acc * g.end() in the gradients' type (OUT: BF16, F16, or 3: fp32).  tokens: n is a token, and
// rows that take no part are 0 (their sums of zeros times an infinite weight or factor are NaN)
template <int OUT>
struct GradEpi {
  static constexpr Ends kEnds{9, 14, OUT == 3};
  struct Args {
    void* out;
    int64_t ld;
    GradOf g;
    int N, M, tokens;
    __device__ __forceinline__ bool live(int n) const { return !tokens || (n < N && g.live(n)); }
  };
  template <class C>
  using Pre = NoPre;
  template <class C>
  static __device__ __forceinline__ void run(Tile<C>& t, const Args& e, const Pre<C>& pre, char* lds) {
    const float f = e.g.end();
    if constexpr (OUT == 3) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        const int n = t.col(j);
        if (n >= e.N) continue;
        const bool live = e.live(n);
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          const int m = t.row(i);
          float* o = static_cast<float*>(e.out) + (int64_t)n * e.ld + m;
          const f4v v = live ? t.acc[i][j] * f : f4v{0, 0, 0, 0};
          if (m + 4 <= e.M) {
            *reinterpret_cast<f4u*>(o) = v;
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (m + k < e.M) o[k] = v[k];
          }
        }
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < C::TN; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        const bool live = e.live(t.col(j));
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          const u2v w = {pack2<OUT>(t.acc[i][j][0] * f, t.acc[i][j][1] * f), pack2<OUT>(t.acc[i][j][2] * f, t.acc[i][j][3] * f)};
          stage4(t, lds, i, j, live ? w : u2v{0, 0});
        }
      }
      __syncthreads();
      store_rows<C>(lds, static_cast<uint16_t*>(e.out), e.ld, t.tn * C::BN, t.tm * C::BM, e.N, e.M);
    }
  }
};

// ---- the rows' kernels ---------------------------------------------------

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int w = 32; w; w >>= 1) x += __shfl_xor(x, w);
  return x;
}

// Rows' statistics and losses from the tiles': R rows to a workgroup, 256 / R lanes to a row
// (many rows: neighbouring lanes read neighbouring rows; one row: all lanes share its tiles).
// total: also the sum (mean: over the rows that count) of the losses, and those rows' number.
// Each workgroup publishes its rows' sum past its XCD's cache and counts itself in (a release); the one
// that arrives last (an acquire) adds them up in order.  A launch of its own for that took 3 us.
template <int R>
__global__ __launch_bounds__(256) void row_stats_k(const float2* __restrict__ partial, int parts, int N, int64_t V,
                                                   const float* __restrict__ tlogit, const int64_t* __restrict__ target,
                                                   int64_t ignore, float k, float lift, float2* __restrict__ stat, float* __restrict__ rest,
                                                   float* __restrict__ loss, double* sums, uint32_t* arrived, int mean,
                                                   float* __restrict__ total, float* __restrict__ count) {
  __shared__ float2 red[256];
  const int row = threadIdx.x % R, n = blockIdx.x * R + row;
  float m = -INFINITY, s = 0.f;
  if (n < N)
    for (int p = threadIdx.x / R; p < parts; p += 8 * (256 / R)) {
      float2 o[8];                                           // loads in flight together: they come from other XCDs
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = p + u * (256 / R);
        o[u] = at < parts ? partial[(int64_t)at * N + n] : make_float2(-INFINITY, 0.f);
      }
      float t = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) t = fmaxf(t, o[u].x);
      const float ref = t == -INFINITY ? 0.f : t;
      s *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
      for (int u = 0; u < 8; ++u) s += o[u].y * __builtin_amdgcn_exp2f(o[u].x - ref);
      m = t;
    }
  red[threadIdx.x] = make_float2(m, s);
  __syncthreads();
#pragma unroll
  for (int w = 128; w >= R; w >>= 1) {
    if (threadIdx.x < w) {
      const float2 a = red[threadIdx.x], b = red[threadIdx.x + w];
      const float t = fmaxf(a.x, b.x), ref = t == -INFINITY ? 0.f : t;
      red[threadIdx.x] = make_float2(t, a.y * __builtin_amdgcn_exp2f(a.x - ref) + b.y * __builtin_amdgcn_exp2f(b.x - ref));
    }
    __syncthreads();
  }
  float l = 0.f;
  bool counts = false;
  if (threadIdx.x < R && n < N) {
    float2 r = red[threadIdx.x];
    const int64_t t = target[n];
    counts = t != ignore;
    // the target's exponent, rounded as it was in its exponential (lift: KeepEpi's): with p next to 1 that rounding
    // would be all of the loss
    float mine = __builtin_fmaf(tlogit[n], k, lift - r.x) - lift;
    if (r.y < 0.5f && r.y > 0.f) {                           // a multiple of a power of two far above the row: nearer to the sum
      const int e = __builtin_amdgcn_frexp_expf(r.y);
      r = make_float2(r.x + e, __builtin_amdgcn_ldexpf(r.y, -e));
      mine -= e;
    }
    stat[n] = make_float2(r.x, 1.f / r.y);
    // 1 - p of the target, from the logit that is in the sum
    rest[n] = counts && t >= 0 && t < V ? 1.f - __builtin_amdgcn_exp2f(mine) * (1.f / r.y) : 0.f;
    // log(sum) - (l_t - max): the maximum leaves before anything is rounded to its size
    l = !counts ? 0.f
        : t < 0 || t >= V ? __uint_as_float(0x7fc00000u)
                          : kLn2 * (__builtin_log2f(r.y) - mine);
    if (loss) loss[n] = l;
  }
  if (!total || threadIdx.x >= 64) return;
  static_assert(R <= 64, "a workgroup's rows in its first wave");
  const double sum = wave_sum(l), num = wave_sum(counts);
  uint32_t order = 0;
  if (threadIdx.x == 0) {
    __hip_atomic_store(sums + 2 * blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(sums + 2 * blockIdx.x + 1, num, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    order = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (__builtin_amdgcn_readfirstlane(order) != gridDim.x - 1) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");         // the other lanes' loads are behind the counter too
  double a = 0, c = 0;
#pragma unroll 4
  for (int b = threadIdx.x; b < gridDim.x; b += 64) {
    a += __hip_atomic_load(sums + 2 * b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    c += __hip_atomic_load(sums + 2 * b + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  a = wave_sum(a);
  c = wave_sum(c);
  if (threadIdx.x == 0) {
    *total = (float)(mean ? a / c : a);
    *count = (float)c;
  }
}

// ratio[n] and *factor (GradOf) of single losses' gradients: relative to the largest finite |g|, so that one that
// is not finite stays its own row's (NaN).  One workgroup: 2.6 us of 40 rows, 9 of 8192, 71 of 65536, 283 of 2^18
// (whose products take 3 ms and more)
__global__ __launch_bounds__(1024) void grad_rows_k(const GradOf g, int N, float* __restrict__ ratio, float* __restrict__ factor) {
  __shared__ float red[1024];
  float top = 0.f;
  for (int n = threadIdx.x; n < N; n += 1024)
    if (g.target[n] != g.ignore && fabsf(g.grad[n]) < INFINITY) top = fmaxf(top, fabsf(g.grad[n]));
  red[threadIdx.x] = top;
  __syncthreads();
  for (int w = 512; w; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + w]);
    __syncthreads();
  }
  top = red[0];
  for (int n = threadIdx.x; n < N; n += 1024) {
    const int64_t t = g.target[n];
    const float x = g.grad[n];
    const bool none = t < 0 || t >= g.V || !(fabsf(x) < INFINITY);
    ratio[n] = t == g.ignore || x == 0.f ? 0.f : none ? __uint_as_float(0x7fc00000u) : x / top * g.lift;
  }
  if (threadIdx.x == 0) *factor = top > 0.f ? top / g.lift * g.c : 0.f;
}

// Eight neighbours of a row as the products take them: 16-bit numbers, or the three bf16 of each fp32.
template <typename T>
struct Eight {
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;
  typedef T v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  i4v plane[P];
  // the first n of p, and zeros
  static __device__ __forceinline__ v8 read(const T* p, int n) {
    v8 v;
    if (n >= 8) {
      v = *reinterpret_cast<const v8*>(p);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = k < n ? p[k] : (T)0;
    }
    return v;
  }
  __device__ __forceinline__ void split(v8 v) {
    if constexpr (P == 3) {
      uint32_t b[3][4] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float f = v[k];
        const bool finite = fabsf(f) < INFINITY;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          uint32_t h = pack2<BF16>(f, 0.f) & 0xffffu;
          // a finite number next to the largest rounds to infinity: cut it off instead
          if ((h & 0x7fffu) == 0x7f80u) h -= 1;
          // infinity and NaN stand in the last plane alone: it meets the other operand's first plane only, so
          // that infinity times a number is infinity (times a zero of its later planes it would be NaN)
          if (!finite) h = q == 2 ? pack2<BF16>(f, 0.f) & 0xffffu : 0;
          b[q][k >> 1] |= h << (16 * (k & 1));
          if (finite) f -= __uint_as_float(h << 16);
        }
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) plane[q] = i4v{(int)b[q][0], (int)b[q][1], (int)b[q][2], (int)b[q][3]};
    } else {
      typedef T w8 __attribute__((ext_vector_type(8)));
      plane[0] = __builtin_bit_cast(i4v, (w8)v);
    }
  }
};

// Rows laid out for the products, cols padded with zeros to a multiple of 8, rows ldo apart, planes behind
// each other.  A thread makes 8 columns.  Two matrices in one launch.
struct PackJob {
  const void* x;
  int64_t ld, rows, plane;
  uint16_t* out;
};
template <typename T>
__global__ __launch_bounds__(256) void pack_k(const PackJob j0, const PackJob j1, int cols, int64_t ldo) {
  const int per = (cols + 7) / 8;
  const int64_t total = (j0.rows + j1.rows) * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const bool second = r >= j0.rows;
    if (second) r -= j0.rows;
    Eight<T> v;
    v.split(v.read(static_cast<const T*>(second ? j1.x : j0.x) + r * (second ? j1.ld : j0.ld) + c, cols - c));
    uint16_t* const o = (second ? j1.out : j0.out) + r * ldo + c;
#pragma unroll
    for (int q = 0; q < Eight<T>::P; ++q) *reinterpret_cast<i4v*>(o + q * (second ? j1.plane : j0.plane)) = v.plane[q];
  }
}

// Rows laid out both ways, from one reading: as pack_k's (rows, if any), and with rows for columns (cols, if
// any): cols[c][r] = x[r][c] for r < Rp (a multiple of 8), zero for r >= R and, masked, for rows that take no part
// (they may hold anything and multiply zeros only).  Two matrices of one width in one launch.  64 rows x 256
// columns to a workgroup, the transpose through LDS as a product's outputs.  fp32, 20011 x 513: 41 us, a
// kernel for each way (the second reading the first's planes) 49.
struct Pane {
  static constexpr int BM = 256, BN = 64, NW = 4;
};
struct LayJob {
  const void* x;
  int64_t ld;
  int R, Rp, masked;
  uint16_t* rows;
  int64_t rplane;
  uint16_t* cols;
  int64_t ldc, cplane;
};
template <typename T>
__global__ __launch_bounds__(256) void lay_k(const LayJob j0, const LayJob j1, int blocks0, int D, int64_t ldr, const GradOf g) {
  __shared__ __attribute__((aligned(16))) char lds[Pane::BM * Pane::BN * 2];
  constexpr int P = Eight<T>::P;
  const bool second = (int)blockIdx.x >= blocks0;
  const LayJob& j = second ? j1 : j0;
  const int r0 = ((int)blockIdx.x - (second ? blocks0 : 0)) * 64, c0 = blockIdx.y * 256;
  const int chunk = threadIdx.x % 32, c = c0 + chunk * 8;
  // one branch over all eight rows, so that their loads are in flight together; rows past the end read the last
  typename Eight<T>::v8 raw[8];
  const T* const x = static_cast<const T*>(j.x) + c;
  if (c + 8 <= D) {
#pragma unroll
    for (int s = 0; s < 8; ++s) raw[s] = Eight<T>::read(x + min(r0 + (int)threadIdx.x / 32 + s * 8, j.R - 1) * j.ld, 8);
  } else {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int r = r0 + threadIdx.x / 32 + s * 8;
      raw[s] = Eight<T>::read(x + min(r, j.R - 1) * j.ld, max(0, D - c));
    }
  }
  Eight<T> v[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int r = r0 + threadIdx.x / 32 + s * 8;
    const bool in = r < j.R && c < D;
    v[s].split(raw[s]);
    if (r >= j.R) {
#pragma unroll
      for (int q = 0; q < P; ++q) v[s].plane[q] = i4v{0, 0, 0, 0};
    }
    if (j.rows && in) {
#pragma unroll
      for (int q = 0; q < P; ++q) *reinterpret_cast<i4v*>(j.rows + q * j.rplane + r * ldr + c) = v[s].plane[q];
    }
    if (j.masked && r < j.R && !g.live(r)) {
#pragma unroll
      for (int q = 0; q < P; ++q) v[s].plane[q] = i4v{0, 0, 0, 0};
    }
  }
  if (!j.cols) return;
#pragma unroll
  for (int q = 0; q < P; ++q) {
    __syncthreads();                                         // the last plane's reads are over
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int n = threadIdx.x / 32 + s * 8;
      *reinterpret_cast<i4v*>(lds + n * 512 + ((chunk ^ turn<Pane>(n)) * 16)) = v[s].plane[q];
    }
    __syncthreads();
    store_columns<Pane>(lds, j.cols + q * j.cplane, j.ldc, r0, c0, j.Rp, D);
  }
}

// The same of fp32 rows as they are: 64 x 64 to a workgroup.
__global__ __launch_bounds__(256) void lay32_k(const LayJob j0, const LayJob j1, int blocks0, int D, int64_t ldr, const GradOf g) {
  __shared__ float tile[64][65];
  const bool second = (int)blockIdx.x >= blocks0;
  const LayJob& j = second ? j1 : j0;
  const int r0 = ((int)blockIdx.x - (second ? blocks0 : 0)) * 64, c0 = blockIdx.y * 64, lane = threadIdx.x % 64, c = c0 + lane;
  const int Dp = (D + 7) / 8 * 8;
  float v[16];
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const int r = r0 + threadIdx.x / 64 + s * 4;
    v[s] = r < j.R && c < D ? static_cast<const float*>(j.x)[r * j.ld + c] : 0.f;
  }
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const int q = threadIdx.x / 64 + s * 4, r = r0 + q;
    if (j.rows && r < j.R && c < Dp) reinterpret_cast<float*>(j.rows)[r * ldr + c] = v[s];
    tile[q][lane] = j.masked && r < j.R && !g.live(r) ? 0.f : v[s];
  }
  if (!j.cols) return;
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const int q = threadIdx.x / 64 + s * 4;
    if (c0 + q < D && r0 + lane < j.Rp) reinterpret_cast<float*>(j.cols)[(c0 + q) * j.ldc + r0 + lane] = tile[lane][q];
  }
}

// four neighbours in the gradients' type (OUT: BF16, F16, or 3: fp32), those below cols; one store, which
// needs no alignment
template <int OUT>
__device__ __forceinline__ void put4(void* out, int64_t at, int cols, f4v v) {
  typedef uint32_t u2u __attribute__((ext_vector_type(2), aligned(2)));
  if constexpr (OUT == 3) {
    float* o = static_cast<float*>(out) + at;
    if (cols >= 4) {
      *reinterpret_cast<f4u*>(o) = v;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < cols) o[k] = v[k];
    }
  } else {
    const u2v w = {pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    if (cols >= 4) {
      *reinterpret_cast<u2u*>(o) = w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < cols) o[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
  }
}

// dh[n][m] = g.end() * the slabs' sum, slab after slab (rows that take no part: 0, as GradEpi's); a thread makes 4 columns
template <int OUT>
__global__ __launch_bounds__(256) void slab_sum_k(const float* __restrict__ slab, int slices, int64_t slice, int64_t ld,
                                                  int N, int M, const GradOf g, void* __restrict__ out, int64_t ldo) {
  const float f = g.end();
  const int per = (int)(ld / 4);
  const int64_t total = (int64_t)N * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / per;
    const int m = (int)(i - n * per) * 4;
    const float* p = slab + n * ld + m;
    f4v v = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const f4v*>(p + s * slice);
    put4<OUT>(out, n * ldo + m, M - m, g.live((int)n) ? v * f : f4v{0, 0, 0, 0});
  }
}

// base[n] = the target's l * log2e, rounded, and 40 (KeepEpi); infinity: the row takes no part; NaN: that
// logit is no number that exponents can be taken against.  A wave to a row.
template <typename T>
__global__ __launch_bounds__(256) void frozen_base_k(const T* __restrict__ h, int64_t ldh, const T* __restrict__ w, int64_t ldw,
                                                     int N, int64_t V, int D, const int64_t* __restrict__ target,
                                                     int64_t ignore, float k, float* __restrict__ base) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= N) return;
  const int64_t t = target[n];
  const bool in = t != ignore && t >= 0 && t < V;
  auto number = [](T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return __uint_as_float((uint32_t)x << 16);
  };
  float sum = 0.f;
  if (in) {
    typedef T v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const T *p = h + n * ldh, *q = w + t * ldw;
    for (int d = lane * 8; d < D; d += 512) {
      if (d + 8 <= D) {
        const v8 x = *reinterpret_cast<const v8*>(p + d), y = *reinterpret_cast<const v8*>(q + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(number(x[i]), number(y[i]), sum);
      } else {
        for (int i = d; i < D; ++i) sum = __builtin_fmaf(number(p[i]), number(q[i]), sum);
      }
    }
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
  sum = __builtin_rintf(sum * k);
  if (lane == 0) base[n] = !in ? INFINITY : fabsf(sum) < INFINITY ? sum + 40.f : __uint_as_float(0x7fc00000u);
}

// A frozen vocabulary's gradient of the embeddings, of an upstream gradient of 1, in fp32:
// dhu[n][m] = c (sum over the slabs of 2^(r - M) / S - (1 - p_t) w[t][m]), with S 2^M the row's
// sum of exponentials; rows that take no part 0, rows whose target is none NaN.  A thread makes 4 columns.
// slab may be dhu itself (one slice): a thread reads the elements that it writes, before it writes them.
template <typename T, bool HALF>
__global__ __launch_bounds__(256) void frozen_dh_k(const float* slab, int slices, int last_slices, int64_t slice,
                                                   int64_t ld, int N, int M, const float* __restrict__ refs,
                                                   const float* __restrict__ refs_before, int64_t ldr, float lift,
                                                   const float2* __restrict__ stat, const float* __restrict__ rests,
                                                   const int64_t* __restrict__ target, int64_t ignore, int64_t V, float c,
                                                   const T* __restrict__ w, int64_t ldw, float* dhu) {
  const int per = (int)(ld / 4);
  const int64_t total = (int64_t)N * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / per;
    const int m = (int)(i - n * per) * 4;
    const int64_t t = target[n];
    f4v v = {0, 0, 0, 0};
    if (t != ignore) {
      const float2 st = stat[n];
      const float* p = slab + n * ld + m;
#pragma unroll 4
      for (int s = 0; s < slices; ++s) {
        // the last piece of the vocabulary may have reached fewer slabs
        const float r = (s < last_slices ? refs : refs_before)[s * ldr + n];
        const float f = r == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r - st.x) * lift;
        v += *reinterpret_cast<const f4v*>(p + s * slice) * f;
      }
      const bool in = t >= 0 && t < V;
      const float rest = in ? rests[n] : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x = 0.f;
        if (in && m + q < M) {
          const T b = w[t * ldw + m + q];
          if constexpr (sizeof(T) == 4) x = b;
          else if constexpr (HALF) x = (float)__builtin_bit_cast(_Float16, b);
          else x = __uint_as_float((uint32_t)b << 16);
        }
        v[q] = c * (v[q] * st.y - rest * x);
      }
    }
    *reinterpret_cast<f4v*>(dhu + n * ld + m) = v;
  }
}

// dh[n][m] = g_n dhu[n][m] (GradOf's rules of rows that take no part)
template <int OUT>
__global__ __launch_bounds__(256) void frozen_scale_k(const float* __restrict__ dhu, int64_t ld, int N, int M,
                                                      const int64_t* __restrict__ target, int64_t ignore,
                                                      const float* __restrict__ grad, int each, const float* __restrict__ count,
                                                      void* __restrict__ out, int64_t ldo) {
  const int per = (int)(ld / 4);
  const int64_t total = (int64_t)N * per;
  const float over = count ? fmaxf(*count, 1.f) : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / per;
    const int m = (int)(i - n * per) * 4;
    const float g = grad[each ? n : 0] / over;
    f4v v = *reinterpret_cast<const f4v*>(dhu + n * ld + m) * g;
    if (target[n] == ignore || g == 0.f) v = f4v{0, 0, 0, 0};
    put4<OUT>(out, n * ldo + m, M - m, v);
  }
}

// ---- few rows ------------------------------------------------------------
// Up to 8 tokens, of fp32 16: the vocabulary's bytes are the work, and one pass over them in their own type, in
// 32-bit arithmetic, makes all of a pass: the logits, then (backward) their part of dh and the rows of dw.
// The products above would read them five times and write two copies (fp32: planes too).
// 8 waves: CW side by side over the columns, 4 to a lane, 256 to a wave; 8 / CW groups of rows.
// A wave holds its columns of all tokens and of their gradients, and R vocabulary rows with
// the next R on their way.  Its R x NB dot products end one to a lane: halves of the values go to
// halves of the lanes, step by step (141 instructions for 64 sums).  The column waves' parts meet
// in LDS, every wave adds them up, and the logits' gradients return as scalars.
// Trained, against the products: 1 x 45459 x 896 fp32 508 -> 98 us (490 MB, 95 us), 1 x 131072 x 2048 bf16
// 739 -> 332, of 8 tokens 519: then it is arithmetic that bounds it, and with 16 tokens of 16 bits the
// matrix cores are quicker (32768 x 1024 bf16 100 us, 146 here; fp32 428, 178 here).
constexpr int kFewRows = 8, kFewRowsF32 = 16, kFewDim = 2048, kFewBlocks = 512;

constexpr int few_batch(int tokens, bool backward) { return tokens <= 8 ? 8 : backward ? 2 : 4; }   // R, as registers allow

template <int M, int STEP>
__device__ __forceinline__ void scatter_sum(float* x, int lane) {
  // M values a lane over lanes that differ in bits STEP and below: the halves go to the lanes without and with that bit
  constexpr int H = M / 2;
  if constexpr (STEP < 0) {
    return;
  } else if constexpr (M == 1) {
    float o;
    if constexpr (STEP >= 4) o = __shfl_xor(x[0], 1 << STEP);
    else if constexpr (STEP == 3) o = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x[0]), 0x140, 15, 15, true));
    else if constexpr (STEP == 2) o = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x[0]), 0x141, 15, 15, true));
    else if constexpr (STEP == 1) o = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x[0]), 0x1b, 15, 15, true));
    else o = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x[0]), 0xb1, 15, 15, true));
    x[0] += o;
    scatter_sum<1, STEP - 1>(x, lane);
  } else {
    // partners: lane ^ 32, ^ 16, then the mirrors of 16, 8, 4 and 2 lanes (the bits below are still alike)
#pragma unroll
    for (int i = 0; i < H; ++i) {
      if constexpr (STEP == 5 || STEP == 4) {
        const auto r = STEP == 5 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + H]), false, false)
                                 : __builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i + H]), false, false);
        x[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      } else {
        const bool high = lane >> STEP & 1;
        const float keep = high ? x[i + H] : x[i], send = high ? x[i] : x[i + H];
        constexpr int ctrl = STEP == 3 ? 0x140 : STEP == 2 ? 0x141 : STEP == 1 ? 0x1b : 0xb1;
        x[i] = keep + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(send), ctrl, 15, 15, true));
      }
    }
    scatter_sum<H, STEP - 1>(x, lane);
  }
}

template <int DT>
struct Row {
  using type = uint16_t;
  static __device__ __forceinline__ float f(uint16_t x) {
    if constexpr (DT == PO_F16) return (float)__builtin_bit_cast(_Float16, x);
    else return __uint_as_float((uint32_t)x << 16);
  }
};
template <>
struct Row<PO_F32> {
  using type = float;
  static __device__ __forceinline__ float f(float x) { return x; }
};

struct FewArgs {
  const void *h, *w;
  int64_t ldh, ldw, V;
  int N, D, cw, batches;        // cw: column waves, 1, 2, 4 or 8
  const int64_t* target;
  int64_t ignore;
  float k;                      // c * log2e
};

// What the two kernels share: a wave's place, its tokens' columns, its rows, their logits.
template <int DT, int NB, int R_>
struct FewWave {
  using T = typename Row<DT>::type;
  typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  static constexpr int R = R_, M = R * NB, SH = M >= 64 ? 0 : M == 32 ? 1 : M == 16 ? 2 : 3;
  static_assert(M <= 64 && M >= 8, "one dot product to a lane at most");
  const FewArgs& a;
  int lane, wave, cwave, group, groups, col, cols;
  float h[NB][4];
  v4 next[R];
  __device__ __forceinline__ explicit FewWave(const FewArgs& args) : a(args) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    cwave = wave % a.cw;
    group = blockIdx.x * (8 / a.cw) + wave / a.cw;
    groups = gridDim.x * (8 / a.cw);
    col = cwave * 256 + lane * 4;
    cols = max(0, min(4, a.D - col));
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        h[n][e] = n < a.N && e < cols ? Row<DT>::f(static_cast<const T*>(a.h)[n * a.ldh + col + e]) : 0.f;
  }
  // the value of this lane after the sums: vocabulary row and token
  __device__ __forceinline__ int my_row() const { return (lane >> SH) / NB; }
  __device__ __forceinline__ int my_token() const { return (lane >> SH) % NB; }
  __device__ __forceinline__ void load(int batch) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t v = (int64_t)batch * R + r;
      const T* p = static_cast<const T*>(a.w) + v * a.ldw + col;
      if (v < a.V && cols == 4) {
        next[r] = *reinterpret_cast<const v4*>(p);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) next[r][e] = v < a.V && e < cols ? p[e] : (T)0;
      }
    }
  }
  // this lane's sum over all columns, h . w
  __device__ __forceinline__ float logit(const float (&w)[R][4], float (*red)[64]) {
    float x[M];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float s = w[r][0] * h[n][0];
#pragma unroll
        for (int e = 1; e < 4; ++e) s = __builtin_fmaf(w[r][e], h[n][e], s);
        x[r * NB + n] = s;
      }
    scatter_sum<M, 5>(x, lane);
    red[wave][lane] = x[0];
    __syncthreads();
    float l = 0.f;
    const int first = wave / a.cw * a.cw;
    for (int c = 0; c < a.cw; ++c) l += red[first + c][lane];
    return l;
  }
};

// partial[block][n] and tlogit as StatsEpi's
template <int DT, int NB>
__global__ __launch_bounds__(512, NB > 4 ? 2 : 4) void few_rows_fwd_k(const FewArgs a, float2* __restrict__ partial, uint32_t* arrived,
                                                         float* __restrict__ tlogit) {
  __shared__ float red[2][8][64];
  __shared__ float2 ends[8][64];
  constexpr int R = few_batch(NB, false);
  FewWave<DT, NB, R> f(a);
  if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
  const int n = f.my_token(), r = f.my_row();
  const int64_t t = n < a.N ? a.target[n] : -1;
  float m = -INFINITY, s = 0.f;
  f.load(f.group);
  const int its = (a.batches + f.groups - 1) / f.groups;
  for (int i = 0; i < its; ++i) {
    float w[R][4];
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[q][e] = Row<DT>::f(f.next[q][e]);
    const int batch = f.group + i * f.groups;
    f.load(batch + f.groups);
    const float x = f.logit(w, red[i & 1]);
    const int64_t v = (int64_t)batch * R + r;
    if (v < a.V) {
      if (v == t && f.cwave == 0) tlogit[n] = x;
      const float y = x * a.k, top = fmaxf(m, y), ref = top == -INFINITY ? 0.f : top;
      s = s * __builtin_amdgcn_exp2f(m - ref) + __builtin_amdgcn_exp2f(y - ref);
      m = top;
    }
  }
  ends[f.wave][f.lane] = make_float2(m, s);
  __syncthreads();
  for (int x = threadIdx.x; x < a.N; x += 512) {
    float2 o = make_float2(-INFINITY, 0.f);
    for (int g = 0; g < 8; g += a.cw)
      for (int q = 0; q < R; ++q) {
        const float2 b = ends[g][(q * NB + x) << f.SH];
        const float top = fmaxf(o.x, b.x), ref = top == -INFINITY ? 0.f : top;
        o = make_float2(top, o.y * __builtin_amdgcn_exp2f(o.x - ref) + b.y * __builtin_amdgcn_exp2f(b.x - ref));
      }
    partial[(int64_t)blockIdx.x * a.N + x] = o;
  }
}

// slab[block][n][ld] (if any): this block's part of dh over c and the upstream gradients' factor; dw (if any)
template <int DT, int NB>
__global__ __launch_bounds__(512, NB > 2 ? 2 : 4) void few_rows_bwd_k(const FewArgs a, const float2* __restrict__ stat, const float* __restrict__ rest, const GradOf g,
                                                                      float* __restrict__ slab, int ld, void* __restrict__ dw,
                                                                      int64_t lddw) {
  __shared__ float red[2][8][64];
  __shared__ float sums[8][256];
  constexpr int R = few_batch(NB, true);
  FewWave<DT, NB, R> f(a);
  constexpr int OUT = DT == PO_F32 ? 3 : DT == PO_F16 ? F16 : BF16;
  const int n = f.my_token(), r = f.my_row();
  const bool in = n < a.N;
  const int64_t t = in ? a.target[n] : -1;
  const float2 st = in ? stat[n] : make_float2(0.f, 0.f);
  const float ratio = in ? g.of_row(n) : 0.f, ir = ratio * st.y, end = g.end();
  // the target's part as the forward pass has it: with p next to 1 the logits' roundings here would be all of it
  const float mine = in ? -rest[n] * ratio : 0.f;
  float dh[NB][4];
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const bool live = q < a.N && g.live(q);                  // rows that take no part may hold anything, NaN too
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dh[q][e] = 0.f;
      if (!live) f.h[q][e] = 0.f;
    }
  }
  f.load(f.group);
  const int its = (a.batches + f.groups - 1) / f.groups;
  for (int i = 0; i < its; ++i) {
    float w[R][4];
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[q][e] = Row<DT>::f(f.next[q][e]);
    const int batch = f.group + i * f.groups;
    f.load(batch + f.groups);
    const float x = f.logit(w, red[i & 1]);
    const int64_t v = (int64_t)batch * R + r;
    float dl = v == t ? mine : __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.k, -st.x)) * ir;
    if (ratio == 0.f || v >= a.V) dl = 0.f;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      f4v out = {0, 0, 0, 0};
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        const float b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dl), (q * NB + y) << f.SH));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dh[y][e] = __builtin_fmaf(b, w[q][e], dh[y][e]);
          out[e] = __builtin_fmaf(b, f.h[y][e], out[e]);
        }
      }
      const int64_t vq = (int64_t)batch * R + q;
      if (dw && vq < a.V && f.cols > 0) put4<OUT>(dw, vq * lddw + f.col, f.cols, out * end);
    }
  }
  if (!slab) return;
#pragma unroll
  for (int y = 0; y < NB; ++y) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[f.wave][f.lane * 4 + e] = dh[y][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.cw * 256 && y < a.N; c += 512) {
      float s = 0.f;
      for (int q = c / 256; q < 8; q += a.cw) s += sums[q][c % 256];
      if (c < ld) slab[((int64_t)blockIdx.x * a.N + y) * ld + c] = s;
    }
  }
}

// dh[n][m] = g.end() * the blocks' sum: 16 groups of 16 threads, 4 columns to a thread, block after block in
// each, then the groups' in order
template <int OUT>
__global__ __launch_bounds__(256) void few_sum_k(const float* __restrict__ slab, int blocks, int64_t slice, int M, const GradOf g,
                                                 void* __restrict__ out, int64_t ldo, int64_t ld) {
  __shared__ f4v part[16][16];
  const int n = blockIdx.y, m = blockIdx.x * 64 + threadIdx.x % 16 * 4, grp = threadIdx.x / 16;
  f4v v = {0, 0, 0, 0};
  if (m < ld) {
    const float* p = slab + n * ld + m;
#pragma unroll 8
    for (int s = grp; s < blocks; s += 16) v += *reinterpret_cast<const f4v*>(p + s * slice);
  }
  part[grp][threadIdx.x % 16] = v;
  __syncthreads();
  if (grp || m >= M) return;
  v = part[0][threadIdx.x];
#pragma unroll
  for (int q = 1; q < 16; ++q) v += part[q][threadIdx.x];
  put4<OUT>(out, n * ldo + m, M - m, g.live(n) ? v * g.end() : f4v{0, 0, 0, 0});
}

// ---- the plan ------------------------------------------------------------

// What a piece of the vocabulary may take of the workspace, its rows laid out, dl and dl^T: 16384 rows of 8192
// tokens.  Beside it stand what does not depend on the piece, h^T and the slabs of dh (8192 x 131072 x 2048 bf16:
// 683 MiB in all, 65536 tokens 1380).  Pieces of
// 8192, whose gradients would stay in the last-level cache, cost dh more (twice the sums read and
// written: 486 against 430 us for 16384 rows) than they save elsewhere.
constexpr int64_t kPieceBytes = 640LL << 20;

// Rows of the operands made here: a multiple of 128 bytes, and long ones no multiple of 512:
// 256 rows a power of two apart fall on few memory channels (dh of a 16384-row piece
// 473 us with rows of 32768 bytes, 430 us with 384 bytes more; 490 us with 320 more, rows
// that start within a 128-byte line).
inline int64_t padded(int64_t n) {
  const int64_t p = (n + 63) / 64 * 64;
  return p >= 1024 && p % 256 == 0 ? p + 192 : p;
}

struct Shape {
  int64_t N, V, D;
  int dtype;
  bool direct_h, direct_w;      // the caller's rows serve as they are
  Form form;                    // of the products
  int planes() const { return form == TRIPLE ? 3 : 1; }
  int es() const { return form == WHOLE ? 4 : 2; }            // bytes of an operand's element
  int halves() const { return planes() * es() / 2; }          // 16-bit places of a number
  int Dp() const { return (int)((D + 7) / 8 * 8); }     // columns of rows laid out here, zeros past D
  int64_t ldp() const { return padded(Dp()); }
  int64_t Np() const { return (N + 31) / 32 * 32; }
  int64_t ldn() const { return padded(Np()); }
};

inline int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

// A workspace laid out from its base; from a null base only its size is of use.
struct Layout {
  char* base;
  int64_t at = 0;
  explicit Layout(void* b) : base(static_cast<char*>(b)) {}
  template <typename T>
  T* take(int64_t n) {
    T* r = reinterpret_cast<T*>(base + at);
    at += up(n * (int64_t)sizeof(T));
    return r;
  }
};

// Vocabulary rows of a piece, per_row bytes each: pieces of one size, a multiple of
// 256 rows, as few as kPieceBytes allows.
inline int64_t piece_rows(int64_t V, int64_t per_row) {
  const int64_t most = std::min<int64_t>(std::max<int64_t>(kPieceBytes / (per_row > 0 ? per_row : 1) / 256 * 256, 256), 1 << 20);
  const int64_t pieces = (V + most - 1) / most, each = (V + pieces - 1) / pieces;
  return std::min(V, (each + 255) / 256 * 256);
}

// Few rows: whether their kernels take a pass, and their grid.
inline int few_tokens_of(int64_t N) { return N <= 1 ? 1 : N <= 2 ? 2 : N <= 4 ? 4 : N <= 8 ? 8 : 16; }
inline int few_columns(int64_t D) { return D <= 256 ? 1 : D <= 512 ? 2 : D <= 1024 ? 4 : 8; }
inline bool few_rows(const Shape& s) { return s.N <= (s.dtype == PO_F32 ? kFewRowsF32 : kFewRows) && s.D <= kFewDim; }
// forward: 16-bit rows that serve as they are go through the matrix cores at the same rate (32768 x 1024
// bf16 13 us)
inline bool few_rows_forward(const Shape& s) { return few_rows(s) && (s.dtype == PO_F32 || !s.direct_w); }
inline int few_batches(const Shape& s, bool backward) { return (int)ceil_div(s.V, few_batch((int)s.N, backward)); }
inline int few_blocks(const Shape& s, bool backward) {
  return std::min(kFewBlocks, (int)ceil_div(few_batches(s, backward), 8 / few_columns(s.D)));
}

struct FwdWs {
  float2* partial;
  double* sums;
  uint32_t* arrived;
  float* tlogit;
  uint16_t *hp, *wp;
  int64_t piece, bytes;
  int parts;
  FwdWs(const Shape& s, void* b) {
    Layout l(b);
    if (few_rows_forward(s)) {
      piece = s.V;
      parts = few_blocks(s, false);
      partial = l.take<float2>((int64_t)parts * s.N);
      tlogit = l.take<float>(s.N);
      sums = l.take<double>(2 * s.N);
      arrived = l.take<uint32_t>(1);
      hp = wp = nullptr;
      bytes = l.at;
      return;
    }
    const int64_t wrow = s.direct_w ? 0 : s.ldp() * 2 * s.halves();
    piece = wrow ? piece_rows(s.V, wrow) : s.V;
    parts = 0;
    for (int64_t v = 0; v < s.V; v += piece) parts += ceil_div(std::min(piece, s.V - v), 128);
    partial = l.take<float2>((int64_t)parts * s.N);
    tlogit = l.take<float>(s.N);
    sums = l.take<double>(2 * s.N);
    arrived = l.take<uint32_t>(1);
    hp = l.take<uint16_t>(s.direct_h ? 0 : s.N * s.ldp() * s.halves());
    wp = l.take<uint16_t>(piece * wrow / 2);
    bytes = l.at;
  }
};

constexpr int kSlabSlices = 64;

struct BwdWs {
  float *ratio, *factor, *slab;
  uint16_t *hp, *ht, *wp, *wt, *dl, *dlt;
  int64_t piece, ldl, slab_ld, slab_slice, bytes;
  Plan dh_plan;
  bool direct_dh;               // one piece in one slice: dh leaves the product as it is wanted
  BwdWs(const Shape& s, bool dh, bool dw, void* b) {
    Layout l(b);
    if (few_rows(s)) {
      ratio = l.take<float>(s.N);
      factor = l.take<float>(1);
      slab_ld = (s.D + 3) / 4 * 4;
      slab_slice = s.N * slab_ld;
      slab = l.take<float>(dh ? few_blocks(s, true) * slab_slice : 0);
      bytes = l.at;
      return;
    }
    const int P = s.halves();
    const int64_t per = (s.direct_w ? 0 : s.ldp() * 2 * P) + (dh ? (s.N + s.D) * 2 * P : 0) + (dw ? s.Np() * 2 * P : 0);
    piece = piece_rows(s.V, per);
    ldl = padded(piece);
    ratio = l.take<float>(s.N);
    factor = l.take<float>(1);
    hp = l.take<uint16_t>(s.direct_h ? 0 : s.N * s.ldp() * P);
    ht = l.take<uint16_t>(dw ? s.D * s.ldn() * P : 0);
    wp = l.take<uint16_t>(s.direct_w ? 0 : piece * s.ldp() * P);
    wt = l.take<uint16_t>(dh ? s.D * ldl * P : 0);
    dl = l.take<uint16_t>(dh ? s.N * ldl * P : 0);
    dlt = l.take<uint16_t>(dw ? piece * s.ldn() * P : 0);
    slab_ld = (s.D + 3) / 4 * 4;
    slab_slice = s.N * slab_ld;
    // a slice's sums are written and read once: 8 bytes of each at about 4 TB/s
    dh_plan = plan_product(s.D, s.N, (int64_t)ceil_div(ldl * s.es(), 128) * (s.form == TRIPLE ? 6 : 1),
                           SlabEpi::kEnds, s.form, kSlabSlices, slab_slice * 8 / 4e6);
    direct_dh = piece >= s.V && dh_plan.slices == 1;
    slab = l.take<float>(dh && !direct_dh ? dh_plan.slices * slab_slice : 0);
    bytes = l.at;
  }
};

struct FrozenWs {
  float2 *partial, *stat;
  double* sums;
  uint32_t* arrived;
  float *tlogit, *rest, *base, *refs, *slab_refs, *slab;
  uint8_t* other;
  uint16_t *hp, *wp, *wt, *kept;
  int64_t piece, ldk, ldr, ldo, slab_ld, slab_slice, bytes;
  Plan plan;
  FrozenWs(const Shape& s, void* b) {
    Layout l(b);
    const int P = s.planes();
    piece = piece_rows(s.V, (s.direct_w ? 0 : s.ldp() * 2 * P) + (s.N + s.D) * 2 * P);
    ldk = padded(piece);
    ldr = (s.N + 3) / 4 * 4;
    int64_t parts = 0;
    for (int64_t v = 0; v < s.V; v += piece) parts += ceil_div(std::min(piece, s.V - v), 128);
    partial = l.take<float2>(parts * s.N);
    stat = l.take<float2>(s.N);
    tlogit = l.take<float>(s.N);
    sums = l.take<double>(2 * s.N);
    arrived = l.take<uint32_t>(1);
    rest = l.take<float>(s.N);
    base = l.take<float>(s.N);
    refs = l.take<float>(ceil_div(piece, 256) * 2 * ldr);
    ldo = ceil_div(s.N, 32);
    other = l.take<uint8_t>(ceil_div(piece, 256) * 2 * ldo);
    hp = l.take<uint16_t>(s.direct_h ? 0 : s.N * s.ldp() * P);
    wp = l.take<uint16_t>(s.direct_w ? 0 : piece * s.ldp() * P);
    wt = l.take<uint16_t>(s.D * ldk * P);
    kept = l.take<uint16_t>(s.N * ldk * P);
    slab_ld = (s.D + 3) / 4 * 4;
    slab_slice = s.N * slab_ld;
    plan = plan_product(s.D, s.N, (int64_t)ceil_div(ldk * 2, 128) * (P == 3 ? 6 : 1), RefSlabEpi::kEnds, s.form, kSlabSlices,
                        slab_slice * 8 / 4e6);
    slab_refs = l.take<float>(2 * plan.slices * ldr);
    slab = l.take<float>(plan.slices > 1 ? plan.slices * slab_slice : 0);       // one: the gradient's own place
    bytes = l.at;
  }
};

// operand rows [r0, r0 + rows) of the caller's matrix, or of buf where they do not serve as they are
struct Side {
  const void* x;
  int64_t ld;
  bool direct;
  uint16_t* buf;
};
inline Operand rows_of(const Shape& s, const Side& m, int64_t r0, int64_t rows) {
  if (m.direct) return Operand{static_cast<const char*>(m.x) + r0 * m.ld * s.es(), m.ld * s.es(), 0, (int)rows};
  return Operand{reinterpret_cast<char*>(m.buf), s.ldp() * s.es(), rows * s.ldp() * 2, (int)rows};
}
// lays them out there, h's rows (0: not this time) and w's in one launch
inline void pack(const Shape& s, const Side& h, int64_t hrows, const Side& w, int64_t w0, int64_t wrows, hipStream_t st) {
  const int es = s.dtype == PO_F32 ? 4 : 2;
  auto job = [&](const Side& m, int64_t r0, int64_t rows) {
    if (m.direct) rows = 0;
    return PackJob{static_cast<const char*>(m.x) + r0 * m.ld * es, m.ld, rows, rows * s.ldp(), m.buf};
  };
  const PackJob a = job(h, 0, hrows), b = job(w, w0, wrows);
  const int64_t items = (a.rows + b.rows) * (s.Dp() / 8);
  if (!items) return;
  const dim3 grid((unsigned)std::min<int64_t>((items + 255) / 256, 8192));
  if (s.dtype == PO_F32)
    hipLaunchKernelGGL((pack_k<float>), grid, dim3(256), 0, st, a, b, (int)s.D, s.ldp());
  else
    hipLaunchKernelGGL((pack_k<uint16_t>), grid, dim3(256), 0, st, a, b, (int)s.D, s.ldp());
}

// rows [r0, r0 + rows) of the caller's matrix: laid out where they do not serve as they are, and (cols) transposed,
// rows ldc apart, planes D rows apart
inline LayJob lay_job(const Shape& s, const Side& m, int64_t r0, int64_t rows, int64_t rp, int masked, uint16_t* cols, int64_t ldc) {
  return LayJob{static_cast<const char*>(m.x) + r0 * m.ld * (s.dtype == PO_F32 ? 4 : 2), m.ld, (int)rows, (int)rp, masked,
                m.direct ? nullptr : m.buf, rows * s.ldp(), cols, ldc, s.D * ldc};
}
inline void lay(const Shape& s, const LayJob& a, const LayJob& b, const GradOf& g, hipStream_t st) {
  auto blocks = [](const LayJob& j) { return j.rows || j.cols ? ceil_div(j.cols ? j.Rp : j.R, 64) : 0; };
  const int b0 = blocks(a), b1 = blocks(b);
  if (!(b0 + b1)) return;
  const bool whole = s.form == WHOLE;
  hipLaunchKernelGGL((whole ? lay32_k : s.dtype == PO_F32 ? lay_k<float> : lay_k<uint16_t>), dim3(b0 + b1, ceil_div(s.D, whole ? 64 : 256)),
                     dim3(256), 0, st, a, b, b0, (int)s.D, s.ldp(), g);
}

// fp32 of few tokens goes through the fp32 matrix instructions: at less than half the planes' rate, but without
// making planes, which is 10 bytes a number and 6 at each reading for 4 (trained, of 30000 x 1024: 40 tokens
// 406 -> 229 us, 100 506 -> 346, 192 574 -> 485; 256 610 against 582, and 106 both ways of 8000 x 300)
constexpr int kWholeRows = 192;
inline Shape shape_of(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N, int64_t V, int64_t D, bool frozen) {
  const Form form = dtype != PO_F32 ? SINGLE : N <= kWholeRows && !frozen ? WHOLE : TRIPLE;
  const int chunk = 16 / (dtype == PO_F32 ? 4 : 2);
  auto serves = [&](const void* x, int64_t ld) { return form != TRIPLE && D % 8 == 0 && ld % chunk == 0 && (uintptr_t)x % 16 == 0; };
  return Shape{N, V, D, dtype, serves(h, ldh), serves(w, ldw), form};
}

inline int check_shape(const char* what, int64_t N, int64_t V, int64_t D, int dtype, int64_t ldh, int64_t ldw) {
  PO_REQUIRE(dtype == PO_F32 || dtype == PO_F16 || dtype == PO_BF16, "%s: unknown dtype %d", what, dtype);
  PO_REQUIRE(N >= 1 && V >= 1 && D >= 1 && N <= (1 << 21) && V < (1LL << 31) - 256 && D <= (1 << 20),
             "%s: bad sizes (N=%lld V=%lld D=%lld)", what, (long long)N, (long long)V, (long long)D);
  PO_REQUIRE(ldh >= D && ldw >= D && ldh <= (1 << 21) && ldw <= (1 << 21), "%s: bad row strides", what);
  return PO_OK;
}

template <int KIND, int P, class Epi>
inline int launch_planned(const Args& a, const typename Epi::Args& e, Plan p, hipStream_t s, const char* what) {
  if (p.tile == FEW) return launch_product<Few<KIND, P>, Epi>(a, e, p.slices, s, what);
  if constexpr (P == 3)
    if (p.tile == SQUARE) return launch_product<Square<KIND>, Epi>(a, e, p.slices, s, what);
  if constexpr (P == 3 && Epi::kEnds.tall)
    if (p.tile == TALL) return launch_product<Tall<KIND>, Epi>(a, e, p.slices, s, what);
  if constexpr (KIND != F32)
    if (p.tile == LARGE) return launch_product<Large<KIND, P>, Epi>(a, e, p.slices, s, what);
  return launch_product<Mid<KIND, P>, Epi>(a, e, p.slices, s, what);
}

template <class Epi>
inline Plan plan_of(const Args& a, Form form) {
  return plan_product(a.A.rows, a.B.rows, (int64_t)ceil_div(a.kbytes, 128) * (form == TRIPLE ? 6 : 1), Epi::kEnds, form);
}

template <class Epi>
inline int64_t first_part(const Args& a, Form form) {
  return whole_rounds(a.A.rows, a.B.rows, (int64_t)ceil_div(a.kbytes, 128) * (form == TRIPLE ? 6 : 1), Epi::kEnds, form);
}

inline void row_stats(const float2* partial, int parts, const Shape& s, const float* tlogit, const int64_t* target, int64_t ignore,
                      float k, float lift, float2* stat, float* rest, double* sums, uint32_t* arrived, int reduction, float* loss, float* count,
                      hipStream_t st) {
  // total: few workgroups, since each counts itself in (1000 of them: 20 us, 63: 6)
  const int N = (int)s.N, R = reduction ? (N <= 64 ? 1 : N <= 512 ? 4 : 16) : N <= 256 ? 1 : N <= 2048 ? 4 : 16;
  hipLaunchKernelGGL((R == 1 ? row_stats_k<1> : R == 4 ? row_stats_k<4> : row_stats_k<16>), dim3(ceil_div(N, R)), dim3(256), 0, st,
                     partial, parts, N, s.V, tlogit, target, ignore, k, lift, stat, rest, reduction ? nullptr : loss, sums, arrived,
                     reduction == 2, reduction ? loss : nullptr, count);
}

#define PO_TRY(x)             \
  do {                        \
    const int rc_ = (x);      \
    if (rc_ != PO_OK) return rc_; \
  } while (0)

inline FewArgs few_args(const Shape& s, const void* h, int64_t ldh, const void* w, int64_t ldw, const int64_t* target, int64_t ignore,
                        float scale, bool backward) {
  return FewArgs{h, w, ldh, ldw, s.V, (int)s.N, (int)s.D, few_columns(s.D), few_batches(s, backward), target, ignore, scale * kLog2e};
}
template <class Fn>
inline void few_dispatch(int dtype, int nb, Fn fn) {
  auto tokens = [&](auto dt) {
    if (nb == 1) fn(dt, std::integral_constant<int, 1>{});
    else if (nb == 2) fn(dt, std::integral_constant<int, 2>{});
    else if (nb == 4) fn(dt, std::integral_constant<int, 4>{});
    else if (nb == 8) fn(dt, std::integral_constant<int, 8>{});
    else if constexpr (decltype(dt)::value == PO_F32) fn(dt, std::integral_constant<int, 16>{});
  };
  if (dtype == PO_F32) tokens(std::integral_constant<int, PO_F32>{});
  else if (dtype == PO_F16) tokens(std::integral_constant<int, PO_F16>{});
  else tokens(std::integral_constant<int, PO_BF16>{});
}

}  // namespace

extern "C" int po_linear_ce_workspace(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N,
                                      int64_t V, int64_t D, int dh, int dw, int64_t* fwd_bytes, int64_t* bwd_bytes) {
  PO_TRY(check_shape("po_linear_ce_workspace", N, V, D, dtype, ldh, ldw));
  const Shape s = shape_of(h, ldh, w, ldw, dtype, N, V, D, false);
  if (fwd_bytes) *fwd_bytes = FwdWs(s, nullptr).bytes;
  if (bwd_bytes) *bwd_bytes = BwdWs(s, dh != 0, dw != 0, nullptr).bytes;
  return PO_OK;
}

extern "C" int po_linear_ce_fwd(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N, int64_t V,
                                int64_t D, const int64_t* target, int64_t ignore_index, float scale, int reduction,
                                void* workspace, int64_t workspace_bytes, float* stat, float* loss, float* count,
                                po_stream_t stream) {
  PO_TRY(check_shape("po_linear_ce_fwd", N, V, D, dtype, ldh, ldw));
  PO_REQUIRE(h && w && target && workspace && stat && loss && (reduction == 0 || count), "po_linear_ce_fwd: null pointer");
  PO_REQUIRE(reduction >= 0 && reduction <= 2, "po_linear_ce_fwd: unknown reduction %d", reduction);
  PO_REQUIRE(scale > 0.f && scale < INFINITY, "po_linear_ce_fwd: the scale must be positive and finite");
  const Shape s = shape_of(h, ldh, w, ldw, dtype, N, V, D, false);
  const FwdWs ws(s, workspace);
  PO_REQUIRE(workspace_bytes >= ws.bytes, "po_linear_ce_fwd: workspace of %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)ws.bytes);
  const hipStream_t st = po::stream_of(stream);
  if (few_rows_forward(s)) {
    const FewArgs f = few_args(s, h, ldh, w, ldw, target, ignore_index, scale, false);
    few_dispatch(dtype, few_tokens_of(N), [&](auto dt, auto nb) {
      hipLaunchKernelGGL((few_rows_fwd_k<decltype(dt)::value, decltype(nb)::value>), dim3(ws.parts), dim3(512), 0, st, f, ws.partial,
                         ws.arrived, ws.tlogit);
    });
    row_stats(ws.partial, ws.parts, s, ws.tlogit, target, ignore_index, f.k, 0.f, reinterpret_cast<float2*>(stat), stat + 2 * N, ws.sums, ws.arrived,
              reduction, loss, count, st);
    return po::check_launch("po_linear_ce_fwd");
  }
  Args a{};
  a.kbytes = s.Dp() * s.es();
  const Side hs{h, ldh, s.direct_h, ws.hp}, wside{w, ldw, s.direct_w, ws.wp};
  a.B = rows_of(s, hs, 0, N);
  StatsEpi::Args e{ws.partial, ws.arrived, ws.tlogit, target, 0, 0, (int)N, 0, scale * kLog2e};
  for (int64_t v = 0; v < V; v += ws.piece) {
    const int64_t rows = std::min(ws.piece, V - v);
    if (s.form == WHOLE) {
      LayJob hj{};
      if (!v) hj = lay_job(s, hs, 0, N, N, 0, nullptr, 0);
      lay(s, lay_job(s, wside, v, rows, rows, 0, nullptr, 0), hj, GradOf{}, st);
    } else {
      pack(s, hs, v ? 0 : N, wside, v, rows, st);
    }
    const Operand W = rows_of(s, wside, v, rows);
    for (int64_t r = 0, part; r < rows; r += part) {
      a.A = W.from(r);
      part = first_part<StatsEpi>(a, s.form);
      a.A.rows = (int)part;
      e.v0 = v + r;
      e.V = (int)part;
      const Plan p = plan_of<StatsEpi>(a, s.form);
      PO_TRY((dtype == PO_F16    ? launch_planned<F16, 1, StatsEpi>(a, e, p, st, "po_linear_ce_fwd")
               : dtype == PO_BF16 ? launch_planned<BF16, 1, StatsEpi>(a, e, p, st, "po_linear_ce_fwd")
               : s.form == TRIPLE ? launch_planned<BF16, 3, StatsEpi>(a, e, p, st, "po_linear_ce_fwd")
                                  : launch_planned<F32, 1, StatsEpi>(a, e, p, st, "po_linear_ce_fwd")));
      e.tile0 += ceil_div(part, p.tile == LARGE ? 256 : 128);
    }
  }
  row_stats(ws.partial, e.tile0, s, ws.tlogit, target, ignore_index, e.k, 0.f, reinterpret_cast<float2*>(stat), stat + 2 * N, ws.sums, ws.arrived,
            reduction, loss, count, st);
  return po::check_launch("po_linear_ce_fwd");
}

namespace {

template <int KIND, int OUT>
int backward(const Shape& s, const BwdWs& ws, const Side& h, const Side& w, const GradOf& g, float scale,
             const float2* stat, void* dh, int64_t lddh, void* dw, int64_t lddw, hipStream_t st) {
  constexpr int P = OUT == 3 && KIND != F32 ? 3 : 1, es = OUT == 3 ? 4 : 2, ES = KIND == F32 ? 4 : 2;   // bytes outside and of the operands
  const char* what = "po_linear_ce_bwd";
  const int N = (int)s.N, D = (int)s.D;
  const Operand H = rows_of(s, h, 0, N);
  for (int64_t v = 0; v < s.V; v += ws.piece) {
    const int rows = (int)std::min(ws.piece, s.V - v);
    const int rp = (rows + 63) / 64 * 64;
    const Operand W = rows_of(s, w, v, rows);
    // the piece's w, and once h, laid out and the other way round
    LayJob hj{};
    if (!v) hj = lay_job(s, h, 0, N, s.Np(), 1, dw ? ws.ht : nullptr, s.ldn());
    lay(s, lay_job(s, w, v, rows, rp, 0, dh ? ws.wt : nullptr, ws.ldl), hj, g, st);
    Args a{};
    // dl of the piece
    a.B = H;
    a.kbytes = s.Dp() * ES;
    for (int64_t r = 0, part; r < rows; r += part) {
      using E = DlogitsEpi<KIND, P>;
      a.A = W.from(r);
      part = first_part<E>(a, s.form);
      a.A.rows = (int)part;
      const typename E::Args e{stat, g, v + r, N, (int)s.Np(), (int)part, (int)(r + part < rows ? part : rp - r), scale * kLog2e,
                               dh ? ws.dl + r * (ES / 2) : nullptr, dw ? ws.dlt + r * s.ldn() * (ES / 2) : nullptr, ws.ldl, s.ldn(), N * ws.ldl,
                               ws.piece * s.ldn()};
      PO_TRY((launch_planned<KIND, P, E>(a, e, plan_of<E>(a, s.form), st, what)));
    }
    if (dh) {                                                // sums over v of dl[n][v] w[v][d]
      a.A = Operand{reinterpret_cast<char*>(ws.wt), ws.ldl * ES, D * ws.ldl * 2, D};
      a.B = Operand{reinterpret_cast<char*>(ws.dl), ws.ldl * ES, N * ws.ldl * 2, N};
      a.kbytes = rp * ES;
      // the last piece may have fewer steps than slices: the other slabs keep their sums
      const Plan p{ws.dh_plan.tile, std::min(ws.dh_plan.slices, ceil_div(a.kbytes, P == 3 ? 64 : 128)), 0};
      if (ws.direct_dh) {
        const typename GradEpi<OUT>::Args ge{dh, lddh, g, N, D, 1};
        PO_TRY((launch_planned<KIND, P, GradEpi<OUT>>(a, ge, p, st, what)));
      } else {
        const SlabEpi::Args se{ws.slab, ws.slab_ld, ws.slab_slice, N, D, v > 0};
        PO_TRY((launch_planned<KIND, P, SlabEpi>(a, se, p, st, what)));
      }
    }
    if (dw) {                                                // dw[v][d] = sum_n dl[n][v] h[n][d]
      a.A = Operand{reinterpret_cast<char*>(ws.ht), s.ldn() * ES, D * s.ldn() * 2, D};
      a.B = Operand{reinterpret_cast<char*>(ws.dlt), s.ldn() * ES, ws.piece * s.ldn() * 2, rows};
      a.kbytes = (int)s.Np() * ES;
      char* out = static_cast<char*>(dw) + v * lddw * es;
      const typename GradEpi<OUT>::Args ge{out, lddw, g, rows, D, 0};
      PO_TRY((launch_planned<KIND, P, GradEpi<OUT>>(a, ge, plan_of<GradEpi<OUT>>(a, s.form), st, what)));
    }
  }
  if (dh && !ws.direct_dh) {
    const int grid = (int)std::min<int64_t>((N * (ws.slab_ld / 4) + 255) / 256, 8192);
    hipLaunchKernelGGL((slab_sum_k<OUT>), dim3(grid), dim3(256), 0, st, ws.slab, ws.dh_plan.slices, ws.slab_slice, ws.slab_ld,
                       N, D, g, dh, lddh);
  }
  return po::check_launch(what);
}

}  // namespace

extern "C" int po_linear_ce_bwd(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N, int64_t V,
                                int64_t D, const int64_t* target, int64_t ignore_index, float scale, int reduction,
                                const float* stat, const float* count, const float* grad, void* workspace,
                                int64_t workspace_bytes, void* dh, int64_t lddh, void* dw, int64_t lddw,
                                po_stream_t stream) {
  PO_TRY(check_shape("po_linear_ce_bwd", N, V, D, dtype, ldh, ldw));
  PO_REQUIRE(h && w && target && workspace && stat && grad && (reduction != 2 || count), "po_linear_ce_bwd: null pointer");
  PO_REQUIRE(reduction >= 0 && reduction <= 2, "po_linear_ce_bwd: unknown reduction %d", reduction);
  PO_REQUIRE(scale > 0.f && scale < INFINITY, "po_linear_ce_bwd: the scale must be positive and finite");
  PO_REQUIRE((!dh || lddh >= D) && (!dw || lddw >= D), "po_linear_ce_bwd: bad row strides");
  if (!dh && !dw) return PO_OK;
  const Shape s = shape_of(h, ldh, w, ldw, dtype, N, V, D, false);
  const BwdWs ws(s, dh != nullptr, dw != nullptr, workspace);
  PO_REQUIRE(workspace_bytes >= ws.bytes, "po_linear_ce_bwd: workspace of %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)ws.bytes);
  const hipStream_t st = po::stream_of(stream);
  const bool few = few_rows(s);                              // their dl stay in 32 bits
  const GradOf g{grad, count, target, ignore_index, V, reduction == 0, reduction == 2, dtype == PO_F16 && !few ? kF16Lift : 1.f, scale,
                 ws.ratio, ws.factor};
  if (g.each) hipLaunchKernelGGL(grad_rows_k, dim3(1), dim3(1024), 0, st, g, (int)N, ws.ratio, ws.factor);
  const float2* st2 = reinterpret_cast<const float2*>(stat);
  if (few) {
    const FewArgs f = few_args(s, h, ldh, w, ldw, target, ignore_index, scale, true);
    const int blocks = few_blocks(s, true);
    few_dispatch(dtype, few_tokens_of(N), [&](auto dt, auto nb) {
      hipLaunchKernelGGL((few_rows_bwd_k<decltype(dt)::value, decltype(nb)::value>), dim3(blocks), dim3(512), 0, st, f, st2, stat + 2 * N, g,
                         dh ? ws.slab : nullptr, (int)ws.slab_ld, dw, lddw);
    });
    if (dh)
      hipLaunchKernelGGL((dtype == PO_F32 ? few_sum_k<3> : dtype == PO_F16 ? few_sum_k<F16> : few_sum_k<BF16>),
                         dim3(ceil_div(D, 64), (unsigned)N), dim3(256), 0, st, ws.slab, blocks, ws.slab_slice, (int)D, g, dh, lddh,
                         ws.slab_ld);
    return po::check_launch("po_linear_ce_bwd");
  }
  const Side hs{h, ldh, s.direct_h, ws.hp}, wside{w, ldw, s.direct_w, ws.wp};
  if (dtype == PO_F16) return backward<F16, F16>(s, ws, hs, wside, g, scale, st2, dh, lddh, dw, lddw, st);
  if (dtype == PO_BF16) return backward<BF16, BF16>(s, ws, hs, wside, g, scale, st2, dh, lddh, dw, lddw, st);
  if (s.form == WHOLE) return backward<F32, 3>(s, ws, hs, wside, g, scale, st2, dh, lddh, dw, lddw, st);
  return backward<BF16, 3>(s, ws, hs, wside, g, scale, st2, dh, lddh, dw, lddw, st);
}

namespace {

template <int KIND, int P>
int frozen_forward(const Shape& s, const FrozenWs& ws, const Side& h, const Side& w, const int64_t* target, float k, const float* base,
                   float* slab, int* parts, int* last_slices, int* pieces, hipStream_t st) {
  const char* what = "po_linear_ce_frozen_fwd";
  const int N = (int)s.N, D = (int)s.D;
  StatsEpi::Args e{ws.partial, ws.arrived, ws.tlogit, target, 0, 0, N, 0, k};
  *pieces = 0;
  for (int64_t v = 0; v < s.V; v += ws.piece, ++*pieces) {
    const int rows = (int)std::min(ws.piece, s.V - v), rp = (rows + 63) / 64 * 64;
    LayJob hj{};
    if (!v) hj = lay_job(s, h, 0, N, N, 0, nullptr, 0);
    lay(s, lay_job(s, w, v, rows, rp, 0, ws.wt, ws.ldk), hj, GradOf{}, st);
    const Operand W = rows_of(s, w, v, rows);
    Args a{};
    a.B = rows_of(s, h, 0, N);
    a.kbytes = s.Dp() * 2;
    for (int64_t r = 0, part; r < rows; r += part) {
      using E = KeepEpi<KIND, P>;
      a.A = W.from(r);
      part = first_part<E>(a, s.form);
      a.A.rows = (int)part;
      e.v0 = v + r;
      e.V = (int)part;
      const Plan p = plan_of<E>(a, s.form);
      const typename E::Args ke{e, base, ws.refs + r / 128 * ws.ldr, ws.other + r / 128 * ws.ldo, ws.ldr, ws.ldo,
                                (int)(r + part < rows ? part : rp - r), ws.kept + r, ws.ldk, N * ws.ldk};
      PO_TRY((launch_planned<KIND, P, E>(a, ke, p, st, what)));
      e.tile0 += ceil_div(part, p.tile == LARGE ? 256 : 128);
    }
    a.A = Operand{reinterpret_cast<char*>(ws.wt), ws.ldk * 2, D * ws.ldk * 2, D};
    a.B = Operand{reinterpret_cast<char*>(ws.kept), ws.ldk * 2, N * ws.ldk * 2, N};
    a.kbytes = rp * 2;
    const int64_t half = ws.plan.slices * ws.ldr;
    const Plan p{ws.plan.tile, std::min(ws.plan.slices, ceil_div(a.kbytes, P == 3 ? 64 : 128)), 0};
    const RefSlabEpi::Args se{ws.refs, base, ws.other, ws.ldr, ws.ldo, ceil_div(rp, 128), slab, ws.slab_ld, ws.slab_slice, N, D, v ? ws.slab_refs + (*pieces + 1) % 2 * half : nullptr,
                              ws.slab_refs + *pieces % 2 * half};
    PO_TRY((launch_planned<KIND, P, RefSlabEpi>(a, se, p, st, what)));
    *last_slices = p.slices;
  }
  *parts = e.tile0;
  return PO_OK;
}

}  // namespace

extern "C" int po_linear_ce_frozen_workspace(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N,
                                             int64_t V, int64_t D, int64_t* bytes) {
  PO_TRY(check_shape("po_linear_ce_frozen_workspace", N, V, D, dtype, ldh, ldw));
  PO_REQUIRE(bytes, "po_linear_ce_frozen_workspace: null pointer");
  *bytes = FrozenWs(shape_of(h, ldh, w, ldw, dtype, N, V, D, true), nullptr).bytes;
  return PO_OK;
}

extern "C" int po_linear_ce_frozen_fwd(const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype, int64_t N, int64_t V,
                                       int64_t D, const int64_t* target, int64_t ignore_index, float scale, int reduction,
                                       void* workspace, int64_t workspace_bytes, float* loss, float* count, float* dhu,
                                       po_stream_t stream) {
  PO_TRY(check_shape("po_linear_ce_frozen_fwd", N, V, D, dtype, ldh, ldw));
  PO_REQUIRE(h && w && target && workspace && loss && dhu && (reduction == 0 || count), "po_linear_ce_frozen_fwd: null pointer");
  PO_REQUIRE((uintptr_t)dhu % 16 == 0, "po_linear_ce_frozen_fwd: dhu must start on 16 bytes");
  PO_REQUIRE(reduction >= 0 && reduction <= 2, "po_linear_ce_frozen_fwd: unknown reduction %d", reduction);
  PO_REQUIRE(scale > 0.f && scale < INFINITY, "po_linear_ce_frozen_fwd: the scale must be positive and finite");
  const Shape s = shape_of(h, ldh, w, ldw, dtype, N, V, D, true);
  const FrozenWs ws(s, workspace);
  PO_REQUIRE(workspace_bytes >= ws.bytes, "po_linear_ce_frozen_fwd: workspace of %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)ws.bytes);
  const hipStream_t st = po::stream_of(stream);
  const Side hs{h, ldh, s.direct_h, ws.hp}, wside{w, ldw, s.direct_w, ws.wp};
  const float k = scale * kLog2e;
  float* slab = ws.plan.slices > 1 ? ws.slab : dhu;
  // Its launch costs the host 3 us (500 x 8000 x 384, all the call 72 us or 75) and spares a fifth of
  // the second product's time: from some 25 us of that on.
  const float* base = dtype != PO_F16 && (double)N * V * D * (s.planes() == 3 ? 6 : 1) >= 0x1p34 ? ws.base : nullptr;
  const dim3 rows4(ceil_div(N, 4));
  if (base && dtype == PO_BF16)
    hipLaunchKernelGGL((frozen_base_k<uint16_t>), rows4, dim3(256), 0, st, static_cast<const uint16_t*>(h), ldh,
                       static_cast<const uint16_t*>(w), ldw, (int)N, V, (int)D, target, ignore_index, k, ws.base);
  if (base && dtype == PO_F32)
    hipLaunchKernelGGL((frozen_base_k<float>), rows4, dim3(256), 0, st, static_cast<const float*>(h), ldh,
                       static_cast<const float*>(w), ldw, (int)N, V, (int)D, target, ignore_index, k, ws.base);
  int parts = 0, last = 0, pieces = 0;
  PO_TRY((dtype == PO_F16    ? frozen_forward<F16, 1>(s, ws, hs, wside, target, k, base, slab, &parts, &last, &pieces, st)
          : dtype == PO_BF16 ? frozen_forward<BF16, 1>(s, ws, hs, wside, target, k, base, slab, &parts, &last, &pieces, st)
                             : frozen_forward<BF16, 3>(s, ws, hs, wside, target, k, base, slab, &parts, &last, &pieces, st)));
  row_stats(ws.partial, parts, s, ws.tlogit, target, ignore_index, k, dtype == PO_F16 ? KeepEpi<F16, 1>::kLift : 0.f, ws.stat, ws.rest, ws.sums, ws.arrived, reduction, loss, count, st);
  const int64_t half = ws.plan.slices * ws.ldr;
  const float *refs = ws.slab_refs + (pieces - 1) % 2 * half, *before = ws.slab_refs + pieces % 2 * half;
  const int grid = (int)std::min<int64_t>((N * (ws.slab_ld / 4) + 255) / 256, 8192);
  const float lift = dtype == PO_F16 ? 0x1p-15f : 1.f;
#define PO_DH(T, HALF)                                                                                                     \
  hipLaunchKernelGGL((frozen_dh_k<T, HALF>), dim3(grid), dim3(256), 0, st, slab, ws.plan.slices, last, ws.slab_slice, ws.slab_ld, \
                     (int)N, (int)D, refs, before, ws.ldr, lift, ws.stat, ws.rest, target, ignore_index, V, scale,     \
                     static_cast<const T*>(w), ldw, dhu)
  if (dtype == PO_F32) PO_DH(float, false);
  else if (dtype == PO_F16) PO_DH(uint16_t, true);
  else PO_DH(uint16_t, false);
#undef PO_DH
  return po::check_launch("po_linear_ce_frozen_fwd");
}

extern "C" int po_linear_ce_frozen_bwd(const float* dhu, int dtype, int64_t N, int64_t D, const int64_t* target,
                                       int64_t ignore_index, int reduction, const float* count, const float* grad, void* dh,
                                       int64_t lddh, po_stream_t stream) {
  PO_TRY(check_shape("po_linear_ce_frozen_bwd", N, 1, D, dtype, D, D));
  PO_REQUIRE(dhu && target && grad && dh && (reduction != 2 || count), "po_linear_ce_frozen_bwd: null pointer");
  PO_REQUIRE((uintptr_t)dhu % 16 == 0, "po_linear_ce_frozen_bwd: dhu must start on 16 bytes");
  PO_REQUIRE(reduction >= 0 && reduction <= 2, "po_linear_ce_frozen_bwd: unknown reduction %d", reduction);
  PO_REQUIRE(lddh >= D, "po_linear_ce_frozen_bwd: bad row strides");
  const hipStream_t st = po::stream_of(stream);
  const int64_t ld = (D + 3) / 4 * 4;
  const int grid = (int)std::min<int64_t>((N * (ld / 4) + 255) / 256, 8192);
  hipLaunchKernelGGL((dtype == PO_F32    ? frozen_scale_k<3>
                      : dtype == PO_F16 ? frozen_scale_k<F16>
                                        : frozen_scale_k<BF16>),
                     dim3(grid), dim3(256), 0, st, dhu, ld, (int)N, (int)D, target, ignore_index, grad, reduction == 0,
                     reduction == 2 ? count : nullptr, dh, lddh);
  return po::check_launch("po_linear_ce_frozen_bwd");
}
