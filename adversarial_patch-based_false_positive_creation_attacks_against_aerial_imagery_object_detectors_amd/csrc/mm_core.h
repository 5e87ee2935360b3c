// The matrix-product core of the large-vocabulary head (vocab_loss.hip,
// int8_ops.hip): C[m][n] = sum_k A[m][k] * B[n][k], both operands with k
// contiguous, 16-bit floats, 8-bit integers or fp32 (as it is, or as three planes of
// bf16: product3), sums in 32 bits.
//
// One form only.  LDS reads with a transpose (ds_read_b64_tr_b16) run at 64 B
// per clock and CU against 128 B for plain 16-byte reads (measured 41 against
// 84 TB/s over the chip), and a product of two 256-row tiles already needs
// three quarters of the latter; so operands that a product needs the other way
// round are written that way once (a transpose, or the epilogue that makes
// them), and every product runs this loop.
//
// A workgroup owns a BM x BN tile, its waves WM x WN rectangles of 16 x 16 MFMA
// blocks (v_mfma 16x16x32 of 16-bit floats, 16x16x64 of bytes, 16x16x4 of fp32).  k advances in steps
// of KB bytes per row; STAGES LDS buffers are filled ahead by 16-byte LDS-DMA.  Rows
// are KB bytes, their 16-byte chunks XOR-swizzled by row (by the address each lane
// loads from: the DMA writes LDS linearly), so 8 neighbouring lanes' fragment reads
// cover all banks.  Rows past the operand's end and k past its length read as zero
// (out-of-range buffer offsets).
//
// What bounds it, of a long k, is the chip's power: an 8192^3 bf16 product takes a quarter less time on
// zeros than on random numbers (clock 1.9 to 2.1 GHz, matrix cores 55 % busy).  So the
// form that moves least wins.  Of a short k it is the tiles' ends as well, which a LARGE tile, alone on
// its CU, leaves uncovered: a round of the losses' tiles takes 33.7 us of 16 steps and 52 of 32, so some 15 us
// of each are the first loads and the epilogue.  At 8192^3, fp32 outputs: 8 waves of 128 x 64 in
// 32x32x16 blocks 1.07 ms; in 16x16x32 blocks, which read and write accumulators half as
// often, 0.91; 4 waves of 128 x 128 0.99 and 0.86 (a third less read from LDS), but a wave
// alone on its SIMD leaves the epilogues uncovered: the losses' forward product of
// 131072 x 8192 x 2048 takes 3.28 ms (1340 TFLOP/s) with 8 waves and 3.64 with 4.
// Fragments are read one group ahead, a read behind every second MFMA (6 % over the
// compiler's order); MFMAs go through a wave's blocks to and fro, so that one operand of each is
// the last one's (8192 x 131072 x 2048, trained: 14.45 -> 14.32 ms).
#pragma once
#include "common.h"
#include <algorithm>
#include <type_traits>

namespace po {
namespace mm {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // in memory, wherever it starts
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

enum Kind { BF16 = 0, F16 = 1, I8 = 2, F32 = 3 };

template <int KIND>
struct Acc {
  using type = f4v;
};
template <>
struct Acc<I8> {
  using type = i4v;
};

template <int KIND>
__device__ __forceinline__ typename Acc<KIND>::type mfma(i4v a, i4v b, typename Acc<KIND>::type c) {
  if constexpr (KIND == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  else if constexpr (KIND == F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  else if constexpr (KIND == I8)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  else {
    // four products of 4 k; which k stands in which place of a chunk is the same in both operands
    const f4v x = __builtin_bit_cast(f4v, a), y = __builtin_bit_cast(f4v, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[k], y[k], c, 0, 0, 0);
    return c;
  }
}

// One operand: rows of k-contiguous elements, stride and length in bytes (both
// multiples of 16 where they are read: the host pads or refuses others).
struct Operand {
  const char* p;
  int64_t stride;   // bytes from row to row (256 rows stay under 2 GiB)
  int64_t plane;    // bytes from plane to plane (operands split into planes)
  int rows;
  Operand from(int64_t r) const { return Operand{p + r * stride, stride, plane, (int)(rows - r)}; }
};

constexpr uint32_t kOOB = 0x80000000u;

template <int KIND_, int BM_, int BN_, int WM_, int WN_, int KB_, int STAGES_, int KG_ = 1, int PLANES_ = 1>
struct Cfg {
  static constexpr int KG = KG_;                                         // groups of waves that take k-steps in turn
  static constexpr int PLANES = PLANES_;                                 // 3: a step holds both operands' three (product3)
  static constexpr int KIND = KIND_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, KB = KB_, STAGES = STAGES_;
  static constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  static constexpr int RPI = 1024 / KB;                                  // rows one wave's DMA instruction fills
  static constexpr int NA = (BM / RPI + NW - 1) / NW, NB = (BN / RPI + NW - 1) / NW;   // instructions per wave and stage
  static constexpr int STAGE_BYTES = (BM + BN) * KB * PLANES, LDS = KG * STAGES * STAGE_BYTES;
  static_assert(KB % 64 == 0 && BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && BM % RPI == 0 && BN % RPI == 0, "tile");
  static_assert(PLANES == 3 || (NA * RPI * NW == BM && NB * RPI * NW == BN), "every wave loads as much");
  static_assert((KG - 1) * BM * BN * 4 <= LDS, "the groups' sums pass through LDS");
};

template <int KB>
__device__ __forceinline__ int swz(int row) {
  return KB == 256 ? (row & 15) : (row & 7);
}

template <class C>
struct Loader {
  __amdgpu_buffer_rsrc_t rs;
  static __device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t rs, char* lds, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
  }
};

// B may hold, in place of numbers, their multiples by powers of two that differ from one 128 of k to the
// next (a block): those of block b in row n are 2^-r times the numbers, r = ref[b][n] a whole number
// (-infinity: all zero).  Refs keeps the sums of a column as multiples of 2^-(the last block's r): where r
// changes the sums are multiplied by 2^(old - new), exactly.  A block whose r lies 48 below
// the column's largest so far is left out: its numbers are below 2^-48 of that block's largest
// one, and sums that followed r downwards without end would overflow.  A tile's references
// come to LDS by the loads that bring its operands.
struct NoRefs {
  static constexpr bool on = false;
};
template <class C>
struct Refs {
  static constexpr bool on = true;
  static constexpr int SLOTS = 2, COLS = C::TN * 16;
  static constexpr int LDS = SLOTS * 1024 + C::NW * COLS * 8;
  static_assert(C::KG == 1 && C::BN <= 256, "one group's sums, a tile's references in one load");
  const char* p;                                             // of block 0 and the tile's first column
  int64_t ld;                                                // bytes from block to block
  int cols;                                                  // columns there
  char* lds;
  int wave, wn, lane;
  int issued = 0, taken = 0;
  uint32_t left_out = 0;                                     // bit j: this lane's column j of the block
  bool any = false;                                          // some lane's
  // this wave's columns: r of the sums, then the largest so far (in LDS: LARGE has no registers left)
  __device__ __forceinline__ float* state() const { return reinterpret_cast<float*>(lds + SLOTS * 1024) + wave * COLS * 2; }
  __device__ __forceinline__ float last(int j) const { return state()[j * 16 + (lane & 15)]; }
  __device__ __forceinline__ void start() {
    for (int i = lane; i < COLS * 2; i += 64) state()[i] = -INFINITY;
  }
  __device__ __forceinline__ void load(int block) {
    if (wave == 0) {
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p + block * ld), 0, 0x7fffffff, 0x00020000);
      Loader<C>::dma(rs, lds + (issued % SLOTS) * 1024, lane * 4 < C::BN && lane * 4 < cols ? (uint32_t)lane * 16 : kOOB);
    }
    ++issued;
  }
  static __device__ __forceinline__ float pow2(float d) { return __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(d, -300.f)); }
  __device__ __forceinline__ void take(f4v (&acc)[C::TM][C::TN]) {
    const float* slot = reinterpret_cast<const float*>(lds + (taken % SLOTS) * 1024) + wn * COLS;
    float* st = state();
    ++taken;
    float by[C::TN];
    bool change = false;
    left_out = 0;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int c = j * 16 + (lane & 15);
      const float r = slot[c], old = st[c], top = st[COLS + c];
      const bool out = r == -INFINITY || r < top - 48.f;
      left_out |= (uint32_t)out << j;
      by[j] = out || old == -INFINITY ? 1.f : pow2(old - r);
      change |= by[j] != 1.f;
      if (!out && lane < 16) {
        st[c] = r;
        st[COLS + c] = fmaxf(top, r);
      }
    }
    any = __any(left_out != 0);
    if (__any(change)) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int i = 0; i < C::TM; ++i) acc[i][j] *= by[j];
    }
  }
  __device__ __forceinline__ void mask(i4v (&b)[C::TN]) const {
    if (any) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
        if (left_out >> j & 1) b[j] = i4v{0, 0, 0, 0};
    }
  }
};

// acc += the tile's product over the k-steps [ks0, ks1).  kbytes: length of a row; ends inside a step
// read as zero.  ks1 > ks0.
template <class C, class RefsT>
__device__ __forceinline__ void product(typename Acc<C::KIND>::type (&acc)[C::TM][C::TN], const Operand& A,
                                        const Operand& B, int m0, int n0, int kbytes, int ks0, int ks1, char* lds,
                                        RefsT& refs) {
  constexpr int KB = C::KB, CPR = KB / 16;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wid % C::NW, kg = wid / C::NW;
  lds += kg * C::STAGES * C::STAGE_BYTES;
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int lrow = lane / CPR;                               // row of this lane inside one DMA instruction
  uint32_t oa[C::NA], ob[C::NB];
#pragma unroll
  for (int i = 0; i < C::NA; ++i) {
    const int r = (i * C::NW + wave) * C::RPI + lrow;
    const int ch = (lane % CPR) ^ swz<KB>(r);
    oa[i] = m0 + r < A.rows ? (uint32_t)(r * (int)A.stride) + ch * 16 : kOOB;
  }
#pragma unroll
  for (int i = 0; i < C::NB; ++i) {
    const int r = (i * C::NW + wave) * C::RPI + lrow;
    const int ch = (lane % CPR) ^ swz<KB>(r);
    ob[i] = n0 + r < B.rows ? (uint32_t)(r * (int)B.stride) + ch * 16 : kOOB;
  }
  // the chunk of this lane inside a step is the same in every instruction: rows
  // of one lane differ by multiples of RPI * NW, which the swizzle does not see
  static_assert((C::RPI * C::NW) % (KB == 256 ? 16 : 8) == 0 && (KB == 128 || KB == 256), "swizzle period");
  const uint32_t lch = ((lane % CPR) ^ swz<KB>(wave * C::RPI + lrow)) * 16;
  const char* abase = A.p + (int64_t)m0 * A.stride;
  const char* bbase = B.p + (int64_t)n0 * B.stride;
  int next = ks0 + kg;                                       // the next stage's step
  constexpr int PER = 256 / KB;                              // steps of a block of references
  if constexpr (RefsT::on) refs.start();
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(abase), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(bbase), 0, 0x7fffffff, 0x00020000);
  auto issue = [&](int buf) {
    if constexpr (RefsT::on)
      if (next % PER == 0 || next == ks0) refs.load(next / PER);   // ahead of the operands: the waits below count them
    char* la = lds + buf * C::STAGE_BYTES;
    char* lb = la + C::BM * KB;
    const uint32_t k0 = (uint32_t)next * KB;
    // past the row's end: out of range by the sign bit (offsets stay below 2^31)
    const uint32_t past = (int)(k0 + lch) < kbytes && (C::KG == 1 || next < ks1) ? k0 : kOOB;
#pragma unroll
    for (int i = 0; i < C::NA; ++i)
      Loader<C>::dma(ra, la + (i * C::NW + wave) * 1024, (oa[i] + (past & 0x7fffffffu)) | (past & kOOB) | (oa[i] & kOOB));
#pragma unroll
    for (int i = 0; i < C::NB; ++i)
      Loader<C>::dma(rb, lb + (i * C::NW + wave) * 1024, (ob[i] + (past & 0x7fffffffu)) | (past & kOOB) | (ob[i] & kOOB));
    next += C::KG;
  };
  const int n = (ks1 - ks0 + C::KG - 1) / C::KG;             // of every group: a last step past the end adds zeros
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s)
    if (s < n) issue(s);
  const int ar = wm * C::TM * 16 + (lane & 15), br = wn * C::TN * 16 + (lane & 15), h = lane >> 4;
  constexpr int G = KB / 64;                                 // groups of fragments in a step
  i4v fa[2][C::TM], fb[2][C::TN];
  auto fetch = [&](int buf, int g, i4v (&a)[C::TM], i4v (&b)[C::TN]) {
    const char* la = lds + buf * C::STAGE_BYTES;
    const char* lb = la + C::BM * KB;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int r = br + j * 16;
      b[j] = *reinterpret_cast<const i4v*>(lb + r * KB + (((4 * g + h) ^ swz<KB>(r)) * 16));
    }
#pragma unroll
    for (int i = 0; i < C::TM; ++i) {
      const int r = ar + i * 16;
      a[i] = *reinterpret_cast<const i4v*>(la + r * KB + (((4 * g + h) ^ swz<KB>(r)) * 16));
    }
  };
  auto multiply = [&](const i4v (&a)[C::TM], const i4v (&b)[C::TN]) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int jj = 0; jj < C::TN; ++jj) {
        const int j = i & 1 ? C::TN - 1 - jj : jj;
        acc[i][j] = mfma<C::KIND>(a[i], b[j], acc[i][j]);
      }
    // the next group's reads between these MFMAs
    constexpr int R = C::TM + C::TN, X = C::TM * C::TN * (C::KIND == F32 ? 4 : 1);
    constexpr int E = C::KIND == F32 ? X / R : X >= 2 * R ? 2 : 1;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, E, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, X > E * R ? X - E * R : 0, 0);
  };
  static_assert(G % 2 == 0, "a step's groups alternate between two sets of registers");
  int buf = 0, s = 0;
  auto step = [&](auto first) {
    // this step's loads have landed when at most the later stages' are in flight; the
    // fragments of the step before have left LDS
    if (C::STAGES > 2 && s + C::STAGES - 2 < n)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((C::STAGES - 2) * (C::NA + C::NB)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                            // ... every wave's
    asm volatile("" ::: "memory");
    if (s + C::STAGES - 1 < n) issue(buf == 0 ? C::STAGES - 1 : buf - 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch(buf, 0, fa[0], fb[0]);
    if constexpr (!first) multiply(fa[1], fb[1]);            // the last group of the step before
    if constexpr (RefsT::on) {
      __builtin_amdgcn_sched_barrier(0);
      if (first || (ks0 + s) % PER == 0) refs.take(acc);
      refs.mask(fb[0]);
    }
#pragma unroll
    for (int g = 1; g < G; ++g) {
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (RefsT::on)
        if (g > 1) refs.mask(fb[(g & 1) ^ 1]);
      fetch(buf, g, fa[g & 1], fb[g & 1]);
      multiply(fa[(g & 1) ^ 1], fb[(g & 1) ^ 1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (RefsT::on) refs.mask(fb[1]);
    buf = buf + 1 == C::STAGES ? 0 : buf + 1;
  };
  step(std::true_type{});
  for (s = 1; s < n; ++s) step(std::false_type{});
  multiply(fa[1], fb[1]);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (C::KG > 1) {                                 // the groups' sums, in order, in the first one's registers
    lds -= kg * C::STAGES * C::STAGE_BYTES;
    using V = typename Acc<C::KIND>::type;
    __syncthreads();
    V* sums = reinterpret_cast<V*>(lds) + wave * C::TM * C::TN * 64 + lane;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
        if (kg > 0) sums[(kg - 1) * (C::BM * C::BN / 4) + (i * C::TN + j) * 64] = acc[i][j];
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int g = 0; g < C::KG - 1; ++g)
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
          for (int j = 0; j < C::TN; ++j) acc[i][j] += sums[g * (C::BM * C::BN / 4) + (i * C::TN + j) * 64];
    }
  }
}

// The same of operands in three planes: acc += A0 B0 + A0 B1 + A1 B0 + A1 B1 + A0 B2 + A2 B0.
// A step holds 32 k of all six planes: what product() loads and reads for each of the six
// products is loaded once, and read once into registers (a 64 x 64 wave takes 24 fragments for 96
// MFMAs where the pairs in turn take 36; fp32 head of 3000 x 5000 x 1500, trained: the four
// products 1100 -> 980 us, of 512 x 8192 x 256 126 -> 100).  Rows are 64 bytes, four chunks, turned every four rows:
// of 8 neighbouring lanes' reads every two fall on the same banks (rows 0 and 2, 1 and 3, 4 and 6, 5 and 7), and
// half of LDS's cycles are those conflicts (SQ_LDS_BANK_CONFLICT 1.0e7 of SQ_LDS_IDX_ACTIVE 2.0e7, the products of
// 1000 x 20011 x 513).
template <class C, class RefsT>
__device__ __forceinline__ void product3(f4v (&acc)[C::TM][C::TN], const Operand& A, const Operand& B, int m0, int n0,
                                         int kbytes, int ks0, int ks1, char* lds, RefsT& refs) {
  static_assert(C::KB == 64 && C::PLANES == 3 && C::KG == 1 && C::STAGES == 2, "form");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN, lrow = lane / 4;
  // rows of one lane differ by multiples of 16, which the turn does not see
  const uint32_t lch = (uint32_t)((lane & 3) ^ ((lrow >> 2) & 3)) * 16;
  uint32_t oa[C::NA], ob[C::NB];
#pragma unroll
  for (int i = 0; i < C::NA; ++i) {
    const int r = (i * C::NW + wave) * C::RPI + lrow;
    oa[i] = m0 + r < A.rows ? (uint32_t)(r * (int)A.stride) + lch : kOOB;
  }
#pragma unroll
  for (int i = 0; i < C::NB; ++i) {
    const int r = (i * C::NW + wave) * C::RPI + lrow;
    ob[i] = n0 + r < B.rows ? (uint32_t)(r * (int)B.stride) + lch : kOOB;
  }
  const char* abase = A.p + (int64_t)m0 * A.stride;
  const char* bbase = B.p + (int64_t)n0 * B.stride;
  constexpr int PA = C::BM * 64, PB = C::BN * 64;            // bytes of a plane of a stage
  if constexpr (RefsT::on) refs.start();
  auto issue = [&](int buf, int step) {
    if constexpr (RefsT::on)
      if (step % 4 == 0 || step == ks0) refs.load(step / 4);
    const uint32_t k0 = (uint32_t)step * 64;
    const uint32_t past = (int)(k0 + lch) < kbytes ? k0 : kOOB;
    char* la = lds + buf * C::STAGE_BYTES;
    char* lb = la + 3 * PA;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const __amdgpu_buffer_rsrc_t ra =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(abase + p * A.plane), 0, 0x7fffffff, 0x00020000);
      const __amdgpu_buffer_rsrc_t rb =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(bbase + p * B.plane), 0, 0x7fffffff, 0x00020000);
#pragma unroll
      for (int i = 0; i < C::NA; ++i)
        if (C::NA * C::NW * C::RPI == C::BM || i * C::NW + wave < C::BM / C::RPI)
          Loader<C>::dma(ra, la + p * PA + (i * C::NW + wave) * 1024, (oa[i] + (past & 0x7fffffffu)) | (past & kOOB) | (oa[i] & kOOB));
#pragma unroll
      for (int i = 0; i < C::NB; ++i)
        if (C::NB * C::NW * C::RPI == C::BN || i * C::NW + wave < C::BN / C::RPI)
          Loader<C>::dma(rb, lb + p * PB + (i * C::NW + wave) * 1024, (ob[i] + (past & 0x7fffffffu)) | (past & kOOB) | (ob[i] & kOOB));
    }
  };
  const int h = lane >> 4, r16 = lane & 15, turned = (h ^ ((r16 >> 2) & 3)) * 16 + r16 * 64;
  i4v a0[C::TM], a1[C::TM], a2[C::TM], b0[C::TN], b1[C::TN], b2[C::TN];
  auto fetch_a = [&](int buf, int p, i4v (&a)[C::TM]) {
    const char* la = lds + buf * C::STAGE_BYTES + p * PA + wm * C::TM * 1024 + turned;
#pragma unroll
    for (int i = 0; i < C::TM; ++i) a[i] = *reinterpret_cast<const i4v*>(la + i * 1024);
  };
  auto fetch_b = [&](int buf, int p, i4v (&b)[C::TN]) {
    const char* lb = lds + buf * C::STAGE_BYTES + 3 * PA + p * PB + wn * C::TN * 1024 + turned;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) b[j] = *reinterpret_cast<const i4v*>(lb + j * 1024);
  };
  // a product, the next ones' `reads` reads between its MFMAs
  auto multiply = [&](const i4v (&a)[C::TM], const i4v (&b)[C::TN], auto reads) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
      for (int jj = 0; jj < C::TN; ++jj) {
        const int j = i & 1 ? C::TN - 1 - jj : jj;
        acc[i][j] = mfma<C::KIND>(a[i], b[j], acc[i][j]);
      }
    constexpr int R = decltype(reads)::value, X = C::TM * C::TN, each = X / (R ? R : 1), E = each > 1 ? each / 2 * 2 : 1;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, E, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, X > E * R ? X - E * R : 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  using RA = std::integral_constant<int, C::TM>;
  using RB = std::integral_constant<int, C::TN>;
  using RAB = std::integral_constant<int, C::TM + C::TN>;
  using R0 = std::integral_constant<int, 0>;
  issue(0, ks0);
  int buf = 0, s = ks0;
  auto step = [&](auto first) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // this step's loads; the last one's fragments are out
    __builtin_amdgcn_s_barrier();                                 // ... every wave's
    asm volatile("" ::: "memory");
    if (s + 1 < ks1) issue(buf ^ 1, s + 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_a(buf, 0, a0);
    fetch_b(buf, 0, b0);
    if constexpr (!first) multiply(a1, b1, RAB{});                // the last product of the step before
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (RefsT::on) {
      if (first || s % 4 == 0) refs.take(acc);
      refs.mask(b0);
    }
    fetch_b(buf, 2, b2);
    multiply(a0, b0, RB{});
    if constexpr (RefsT::on) refs.mask(b2);
    fetch_a(buf, 2, a2);
    multiply(a0, b2, RA{});
    fetch_b(buf, 1, b1);
    multiply(a2, b0, RB{});
    if constexpr (RefsT::on) refs.mask(b1);
    fetch_a(buf, 1, a1);
    multiply(a0, b1, RA{});
    multiply(a1, b0, R0{});
    buf ^= 1;
  };
  step(std::true_type{});
  for (s = ks0 + 1; s < ks1; ++s) step(std::false_type{});
  multiply(a1, b1, R0{});
}

// Element e of a 16 x 16 accumulator block lies in row (m) 4 * (lane / 16) + e and column
// (n) lane % 16: a lane's four are consecutive rows of one column.  The kernels below take
// the operand whose index is contiguous in the output (or is reduced over) as A.

struct Args {
  Operand A, B;
  int tiles_m, tiles_n;
  int first;                  // tile of this launch's first workgroup
  int kbytes, nk;             // bytes of a row, k-steps
};

template <class C>
struct Tile {
  typename Acc<C::KIND>::type acc[C::TM][C::TN];
  int m0, n0;                 // first row of A and of B of this wave's rectangle
  int tm, tn;
  int lane, wave, wm, wn;
  __device__ __forceinline__ int col(int j) const { return n0 + j * 16 + (lane & 15); }
  __device__ __forceinline__ int row(int i) const { return m0 + i * 16 + 4 * (lane >> 4); }   // of element 0
};

// Epilogues of products whose B has references (Refs) hold kRefs, and say of a tile's columns whether
// they have any but base.
template <class Epi, class = void>
struct HasRefs : std::false_type {};
template <class Epi>
struct HasRefs<Epi, std::void_t<decltype(Epi::kRefs)>> : std::true_type {};

struct NoPre {
  template <class T, class E>
  __device__ __forceinline__ void load(const T&, const E&) {}
};

// Workgroups of 8 tile rows by all tile columns in turn, an XCD's workgroups
// next to each other: its L2 holds the k-window of the operands they share.
// gridDim.y slices the k-steps.  Epi::run ends the tile; what it reads of a token it reads
// before the loop (Pre): its waves have no others to wait behind.
template <class C, class Epi>
__global__ __launch_bounds__(C::NW * C::KG * 64, C::LDS > 81920 ? 1 : 2) void product_k(const Args a, const typename Epi::Args e) {
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  const int id = a.first + xcd_remap();
  constexpr int GM = 8;                                      // 4 and 16: within 0.5 %
  const int grp = id / (GM * a.tiles_n), first = grp * GM, gm = min(GM, a.tiles_m - first);
  const int r = id - grp * GM * a.tiles_n;
  Tile<C> t;
  t.tm = first + r % gm;
  t.tn = r / gm;
  t.lane = threadIdx.x & 63;
  t.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  t.wm = t.wave % C::NW / C::WN;
  t.wn = t.wave % C::WN;
  t.m0 = t.tm * C::BM + t.wm * C::TM * 16;
  t.n0 = t.tn * C::BN + t.wn * C::TN * 16;
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j) t.acc[i][j] = typename Acc<C::KIND>::type{0, 0, 0, 0};
  typename Epi::template Pre<C> pre;
  pre.load(t, e);
  const int ks0 = (int)((int64_t)blockIdx.y * a.nk / gridDim.y), ks1 = (int)((int64_t)(blockIdx.y + 1) * a.nk / gridDim.y);
  auto multiply = [&](auto& refs) {
    if constexpr (C::PLANES == 3)
      product3<C>(t.acc, a.A, a.B, t.tm * C::BM, t.tn * C::BN, a.kbytes, ks0, ks1, lds, refs);
    else
      product<C>(t.acc, a.A, a.B, t.tm * C::BM, t.tn * C::BN, a.kbytes, ks0, ks1, lds, refs);
  };
  if constexpr (HasRefs<Epi>::value) {
    // tokens of one r in all of these blocks: an ordinary product
    float last[C::TN];
    if (Epi::template plain<C>(t, e)) {
      NoRefs none;
      multiply(none);
#pragma unroll
      for (int j = 0; j < C::TN; ++j) last[j] = t.col(j) < e.N ? e.base[t.col(j)] : 0.f;
    } else {
      __shared__ __attribute__((aligned(1024))) char ref_lds[Refs<C>::LDS];
      const int first_col = t.tn * C::BN;
      Refs<C> refs{reinterpret_cast<const char*>(e.refs + first_col), e.ldr * 4, (int)e.ldr - first_col, ref_lds, t.wave, t.wn, t.lane};
      multiply(refs);
#pragma unroll
      for (int j = 0; j < C::TN; ++j) last[j] = refs.last(j);
    }
    Epi::template run<C>(t, e, pre, last);
    return;
  } else {
    NoRefs none;
    multiply(none);
  }
  // waves of the other groups end here; barriers below wait for the ones that remain
  if (C::KG > 1 && t.wave >= C::NW) return;
  if constexpr (!HasRefs<Epi>::value) Epi::template run<C>(t, e, pre, lds);
}

template <class C, class Epi>
inline int launch_product(Args a, const typename Epi::Args& e, int slices, hipStream_t s, const char* what) {
  a.tiles_m = ceil_div(a.A.rows, C::BM);
  a.tiles_n = ceil_div(a.B.rows, C::BN);
  a.nk = ceil_div(a.kbytes, C::KB);
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles >= (1LL << 31) || slices > 65535 || slices > a.nk || a.A.stride * C::BM >= (1LL << 31) ||
      a.B.stride * C::BN >= (1LL << 31) || a.kbytes < 0) {
    set_error("%s: operand too large", what);
    return PO_EINVAL;
  }
  constexpr int64_t kMost = 1 << 22;                         // of 512 threads: a grid's stay below 2^32
  static_assert(C::NW * C::KG * 64 <= 512, "workgroup");
  for (int64_t at = 0; at < tiles; at += kMost) {
    a.first = (int)at;
    hipLaunchKernelGGL((product_k<C, Epi>), dim3((unsigned)std::min(kMost, tiles - at), slices), dim3(C::NW * C::KG * 64), 0, s, a, e);
  }
  return check_launch(what);
}

// ---- which tile ----------------------------------------------------------
// Three tiles: LARGE 256 x 256 (one workgroup of 8 waves to a CU), MID 128 x 128
// (two of 4 waves), FEW 128 x 32 for few columns or few tiles (two of 4 waves).  The choice is the least time over
// the rounds in which the chip takes the tiles, from what a step of k takes a workgroup
// (us, measured: LARGE 1.7, MID 1.08 with two on the CU) and what its start and its
// epilogue take (the epilogue's; MID's are covered by the other workgroup).  So LARGE is
// taken for long k or cheap epilogues, MID for few tiles and short k: the losses' forward
// product of 32768 x 2048 x 512 78 against 95 us; the gradient of the logits there 117
// against 112 us, at k = 128 73 against 63.  slices > 1 cuts k between workgroups, each
// slice's sums then cost sum_us.  Products of three planes: LARGE 256 x 128, MID 128 x 64, SQUARE
// 128 x 128 (one to a CU: of up to 128 tokens it loads the vocabulary once; logits and their gradient of
// 100 x 30000 x 1024 84 and 94 us with MID, 69 and 77), and TALL
// 192 x 128 for widths that fill 256 badly (the gradients of 20011 x 1000 x 513: 172 and 152 us in
// 768 rows of LARGE tiles, 157 and 141 in 576 of TALL).
enum TileId { FEW, MID, LARGE, SQUARE, TALL };
struct Plan {
  TileId tile;
  int slices;
  double us;
};
struct TileKind {
  TileId id;
  int bm, bn, slots;
  double step, ends;            // ends: share of the epilogue's time
};
// of products of single planes, of three (a step: 64 k of one of the six products), and of fp32 as it is
enum Form { SINGLE, TRIPLE, WHOLE };
constexpr TileKind kTiles[3][5] = {
    {{FEW, 128, 32, 512, 0.45, 0}, {MID, 128, 128, 512, 1.08, 1}, {LARGE, 256, 256, 256, 1.7, 1}, {}, {}},
    {{FEW, 128, 32, 512, 0.35, 0}, {MID, 128, 64, 512, 0.45, 0.5}, {LARGE, 256, 128, 256, 0.73, 0.5},
     {SQUARE, 128, 128, 256, 0.42, 0.5}, {TALL, 192, 128, 256, 0.57, 0.4}},
    {{FEW, 128, 32, 512, 1.2, 0}, {MID, 128, 64, 512, 2.1, 0.5}, {}, {}, {}}};
// What the plan has to know of a product's epilogue: us, and whether its tiles may be TALL
struct Ends {
  double mid, large;
  bool tall;
};
inline Plan plan_product(int64_t M, int64_t N, int64_t steps, Ends ends, Form form = SINGLE, int max_slices = 1, double sum_us = 0) {
  Plan best{LARGE, 1, 1e300};
  for (auto& k : kTiles[form]) {
    if (k.id == TALL && !ends.tall) continue;
    if (!k.bm) continue;
    const int64_t tiles = ((M + k.bm - 1) / k.bm) * ((N + k.bn - 1) / k.bn);
    const double end = k.id == FEW ? 5 : k.ends * (k.id == MID ? ends.mid : ends.large);
    // one slice, or as many as fill the chip half, once or twice
    for (int64_t fill : {(int64_t)1, k.slots / 2 / tiles, k.slots / tiles, 2 * k.slots / tiles}) {
      const int s = (int)std::min<int64_t>(fill, std::min<int64_t>(max_slices, steps / 4));
      if (s < 1 && fill != 1) continue;
      const int n = std::max(s, 1);
      const int64_t rounds = (tiles * n + k.slots - 1) / k.slots;
      const double step = k.slots == 512 && tiles * n <= 256 ? 0.65 * k.step : k.step;   // one to a CU
      const double t = rounds * ((double)((steps + n - 1) / n) * step + end) + n * sum_us;
      if (t < best.us) best = Plan{k.id, n, t};
    }
  }
  return best;
}

// Rows of A (of M) to take first: those of whole rounds of LARGE tiles, where the rest is quicker
// with tiles of its own than as one more round (the losses of 50001 x 2047 x 1000: 6.1 rounds).
inline int64_t whole_rounds(int64_t M, int64_t N, int64_t steps, Ends ends, Form form = SINGLE) {
  const int bm = kTiles[form][2].bm, bn = kTiles[form][2].bn;
  if (!bm) return M;
  const int64_t tn = (N + bn - 1) / bn, full = (M + bm - 1) / bm * tn / 256, first = full * 256 / tn * bm;
  if (first <= 0 || first >= M) return M;
  const double gap = 3;                                      // from one launch to the next
  auto us = [&](int64_t m) { return plan_product(m, N, steps, ends, form).us; };
  return us(first) + us(M - first) + gap < us(M) ? first : M;
}

// ---- outputs -------------------------------------------------------------
// A tile of 16-bit outputs passes through LDS as rows [n][m] and leaves as
// 16-byte pieces of whole rows.  16-byte chunk c of row n lies at chunk
// c ^ turn(n): the 8-byte writes of 16 columns, the 16-byte row reads and the
// transposing reads of 4 rows x 32 bytes each touch every bank evenly.
template <class C>
__device__ __forceinline__ int turn(int n) {
  constexpr int H = C::BM / 16;                 // half the chunks of a row
  return ((n & (H - 1)) << 1) | ((n / H) & 1);
}

typedef uint32_t u2v __attribute__((ext_vector_type(2)));

template <class C>
__device__ __forceinline__ void stage4(const Tile<C>& t, char* lds, int i, int j, u2v four) {
  const int n = t.wn * C::TN * 16 + j * 16 + (t.lane & 15);
  const int c = t.wm * C::TM * 2 + i * 2 + (t.lane >> 5);   // 8 outputs to a chunk, this lane's 4 in one half
  *reinterpret_cast<u2v*>(lds + n * (C::BM * 2) + ((c ^ turn<C>(n)) * 16) + 8 * ((t.lane >> 4) & 1)) = four;
}

// rows [n][m] of the staged tile to out (16-bit, leading dimension ld), n < rows, m < cols; 16 bytes at
// a time wherever the rows start (the stores need no alignment)
template <class C>
__device__ __forceinline__ void store_rows(const char* lds, uint16_t* out, int64_t ld, int n0, int m0, int rows,
                                           int cols) {
  typedef int i4u __attribute__((ext_vector_type(4), aligned(2)));
  constexpr int NC = C::BM / 8, STEPS = C::BN * NC / (C::NW * 64), U = STEPS % 8 == 0 ? 8 : STEPS;
  static_assert(STEPS * C::NW * 64 == C::BN * NC, "whole steps");
  // a thread's chunk is the same in every step, its row advances
  constexpr int ROWS = C::NW * 64 / NC;
  const int c = threadIdx.x % NC, n = threadIdx.x / NC, m = m0 + c * 8;
  uint16_t* o = out + (int64_t)(n0 + n) * ld + m;
  for (int s = 0; s < STEPS; s += U) {
    i4v v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = n + (s + u) * ROWS;
      v[u] = *reinterpret_cast<const i4v*>(lds + r * (C::BM * 2) + ((c ^ turn<C>(r)) * 16));
    }
#pragma unroll
    for (int u = 0; u < U; ++u, o += ROWS * ld) {
      if (n0 + n + (s + u) * ROWS >= rows || m >= cols) continue;
      if (m + 8 <= cols) {
        // past the caches' keeping: the next product's operands stay (dh of 4096x32768x1024 233 -> 219 us)
        __builtin_nontemporal_store(v[u], reinterpret_cast<i4u*>(o));
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (m + k < cols) o[k] = (uint16_t)((uint32_t)v[u][k >> 1] >> (16 * (k & 1)));
      }
    }
  }
}

// the staged tile transposed, rows [m][n] of out: m < cols, n0 + n < rows (a multiple of 8)
template <class C>
__device__ __forceinline__ void store_columns(const char* lds, uint16_t* out, int64_t ld, int n0, int m0, int rows,
                                              int cols) {
  typedef short s4v __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  // a wave's step: 16 columns m by 32 rows n, 8 rows to a group of 16 lanes; its steps go along n
  constexpr int MB = C::BM / 16, NB = C::BN / 32, STEPS = MB * NB / C::NW, U = STEPS % 4 == 0 ? 4 : STEPS;
  static_assert(STEPS * C::NW == MB * NB, "whole steps");
  for (int s = 0; s < STEPS; s += U) {
    u2v two[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = wave * STEPS + s + u;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int nr = (x % NB) * 32 + g * 8 + 4 * k + (i >> 2);
        const int c = (x / NB) * 2 + ((i >> 1) & 1);
        const char* p = lds + nr * (C::BM * 2) + ((c ^ turn<C>(nr)) * 16) + 8 * (i & 1);
        two[u][k] = __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                (__attribute__((address_space(3))) s4v*)(const_cast<char*>(p))));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = wave * STEPS + s + u, m = m0 + (x / NB) * 16 + i, n = n0 + (x % NB) * 32 + g * 8;
      if (m < cols && n < rows)
        *reinterpret_cast<i4v*>(out + (int64_t)m * ld + n) =
            i4v{(int)two[u][0][0], (int)two[u][0][1], (int)two[u][1][0], (int)two[u][1][1]};
    }
  }
}

typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
// two floats rounded to nearest even
template <int KIND>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (KIND == F16)
    return __builtin_bit_cast(uint32_t, h2v{(_Float16)x, (_Float16)y});
  else
    return __builtin_bit_cast(uint32_t, b2v{(__bf16)x, (__bf16)y});
}

}  // namespace mm
}  // namespace po
