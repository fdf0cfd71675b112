// paged.hip - the paged 8-bit K/V cache for gfx950: append with the position
// rotation, read-back, and the attention of new rows over it.
//
// No counterpart in the reference, whose cache is one f32 tensor per sequence
// (layer.rs:219-246).  A pool of pages belongs to many sequences; a page is a
// run of blocks of 32 positions, and a block's codes of one KV head share one
// power-of-two scale for K and one for V:
//   value = code * 2^e,  e = the smallest exponent with max |row value| <= 127 * 2^e.
// A power of two because a block fills row by row in decoding: a row that
// raises the exponent shifts the codes already there (one rounding, half to
// even), the steps lost that way sum to less than one final step, and the scale is
// exact in every later product.
#include "common.h"
#include "../kernel_args.h"

using namespace llmrs;

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBlk = kPagedBlock;

// The words of a launch's sequences: in its arguments or in device memory.
__device__ __forceinline__ int word(const PagedSeqs& s, int i) { return s.ext ? s.ext[i] : s.w[i]; }

struct Seq {
  int item, slot, row0, rows, pos;  // item: the work item's number within the sequence
};
// The sequence of a work item: the last one whose first item is not past it
// (a sequence without items starts where the next one does).
__device__ __forceinline__ Seq find_seq(const PagedSeqs& s, int item) {
  // one value per wave, and so held in scalar registers: the compiler takes what is
  // loaded from either of two places to differ from lane to lane
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  Seq q;
  if (s.n == 1) {
    q.item = item;
    q.slot = uni(s.w[1]);
    q.row0 = uni(s.w[2]);
    q.rows = uni(s.w[3]);
    q.pos = uni(s.w[4]);
    return q;
  }
  int i = -1;
  for (int b = 0; b < s.n; b += LLMRS_WAVE) {
    const int l = b + lane_id();
    i += __popcll(__ballot(l < s.n && word(s, l < s.n ? l : 0) <= item));
  }
  i = uni(i);
  const int at = s.n + 4 * i;
  q.item = item - uni(word(s, i));
  q.slot = uni(word(s, at));
  q.row0 = uni(word(s, at + 1));
  q.rows = uni(word(s, at + 2));
  q.pos = uni(word(s, at + 3));
  return q;
}

// The pool block that holds block `b` of a slot, the same for all lanes.  The table is
// read through the scalar cache: a vector load would be waited for together with the
// codes that are on their way (no kernel here writes the table that it reads).
__device__ __forceinline__ int pool_block(const PagedPool& p, int slot, int b) {
  const int* at = p.table + (size_t)slot * p.stride + (b >> p.shift);
  const int page = *(const __attribute__((address_space(4))) int*)(uintptr_t)at;
  return (page << p.shift) + (b & ((1 << p.shift) - 1));
}

// The smallest e in [kPagedExpMin, kPagedExpMax] with amax <= 127 * 2^e: amax =
// f * 2^x with f in [1/2, 1), and 127 = 127/128 * 2^7.
__device__ __forceinline__ int needed_exp(double amax) {
  amax = fmin(amax, 340282366920938463463374607431768211456.0);  // 2^128: infinities
  const int e = __builtin_amdgcn_frexp_exp(amax) - 7 + (__builtin_amdgcn_frexp_mant(amax) > 127.0 / 128.0 ? 1 : 0);
  return amax > 0.0 ? min(max(e, kPagedExpMin), kPagedExpMax) : kPagedExpMin;
}

// c * 2^-d to the nearest integer, half to even, for 0 <= d <= 8.
__device__ __forceinline__ int shift_code(int c, int d) {
  return d ? (c + ((1 << (d - 1)) - 1) + ((c >> d) & 1)) >> d : c;
}

// The code of a value: the nearest integer, half to even.  The conversions of the
// hardware take NaN to 0 and what is too large to the ends of the range, which C++
// leaves open.
__device__ __forceinline__ int code_of(float x, int e) {
  int c;
  asm("v_cvt_i32_f32 %0, %1" : "=v"(c) : "v"(rintf(ldexpf(x, -e))));
  return min(max(c, -127), 127);
}
__device__ __forceinline__ int code_of(double x, int e) {
  int c;
  asm("v_cvt_i32_f64 %0, %1" : "=v"(c) : "v"(rint(ldexp(x, -e))));
  return min(max(c, -127), 127);
}

// A word of four older codes, rounded to a step 2^d times theirs.
__device__ __forceinline__ unsigned shift_word(unsigned w, int d, int bias) {
  unsigned out = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    out |= ((unsigned)(shift_code((int)(int8_t)((w >> (8 * b)) ^ (unsigned)bias), d) + bias) & 255u) << (8 * b);
  return out;
}
// Bytes [0, n) of the one, the others of the other (n may be any number).
__device__ __forceinline__ unsigned first_bytes(unsigned w, unsigned other, int n) {
  const unsigned mask = n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
  return (w & mask) | (other & ~mask);
}

// Threads for a block of 32 positions of one KV head, K or V.
constexpr int block_threads(int hd) { return 2 * hd; }

}  // namespace

// Appends rows to one block of one sequence.  A thread has 16 codes, and so nobody else
// writes its bytes: of V a dim's 16 positions, of K four dims and their rotation
// partners at two positions.  All its rows are asked for before the first is looked at.
// Older codes are loaded and, where the new rows raise the exponent, rounded to the
// new step.  K is rotated in 64 bits (the products of f32 values are exact there), so
// a code does not depend on how a sum was rounded.
// Bound by memory for prompts: 4 x 2048 rows of 8 heads x 128 in 20.5 us (median of 125
// launches; the fastest 18.7), 84 MB at 4.1 to 4.5 TB/s (a copy reaches 5.1); with the
// codes passed through LDS byte by byte the fastest was about 25.  A decode step of 64
// sequences takes 5.1 us and one row 3.3, a chain of
// dependent accesses (words, page, exponent, codes); 64-bit work where no new row is made
// it 6.8.
template <int HD>
__device__ __forceinline__ void append_block(const PagedRowsArgs& a) {
  constexpr int MID = HD / 2, BYTES = kBlk * HD, LANES = MID / 4, WAVES = block_threads(HD) / LLMRS_WAVE;
  __shared__ float red[WAVES];
  const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
  const Seq q = find_seq(a.seqs, blockIdx.x);
  const int block = q.pos / kBlk + q.item;                  // of the sequence
  const int old = max(0, q.pos - block * kBlk);             // rows already there
  const int end = min(kBlk, q.pos + q.rows - block * kBlk); // rows after
  const size_t unit = ((size_t)pool_block(a.pool, q.slot, block) * a.pool.nkv + head) * 2 + which;
  uint8_t* dst = a.pool.codes + unit * BYTES;
  const int row0 = q.row0 + block * kBlk - q.pos;  // row of the block's position 0
  // (a position without a new row: the nearest that has one)
  auto near = [&](int p) { return min(max(p, old), end - 1); };
  const float* src = a.rows[which] + (size_t)head * HD;
  auto row = [&](int p) { return src + (size_t)(row0 + near(p)) * (a.pool.nkv * HD); };
  auto exponent = [&](double amax) {  // of the block, from every thread's largest magnitude
    float e = wave_max((float)needed_exp(amax));
    if (lane_id() == 0) red[wave_id()] = e;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) e = fmaxf(e, red[w]);
    return (int)e;
  };
  const int e_old = old ? a.pool.exps[unit] : kPagedExpMin;
  int e;
  if (which) {
    const int d = tid % HD, p0 = __builtin_amdgcn_readfirstlane(tid / HD * 16);
    u32x4* at = (u32x4*)(dst + paged_v_offset(p0, d));
    const bool adds = max(old, p0) < min(end, p0 + 16), has = old > p0;
    float x[16] = {}, amax = 0.0f;
    u32x4 was = {0, 0, 0, 0};
    if (has) was = *at;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (p0 + i >= old && p0 + i < end) x[i] = row(p0 + i)[d];
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));  // passes over NaN
    e = max(e_old, exponent(amax));
    if (has && e > e_old)
#pragma unroll
      for (int k = 0; k < 4; ++k) was[k] = shift_word(was[k], min(e - e_old, 8), 128);
    if (adds)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) w |= (unsigned)(code_of(x[4 * k + b], e) + 128) << (8 * b);
        was[k] = first_bytes(was[k], w, old - p0 - 4 * k);
      }
    if (adds || has) *at = was;
  } else {
    constexpr int ROWS = LLMRS_WAVE / LANES;  // of a wave, twice
    const int d = 4 * (tid % LANES), p0 = tid / LANES, first = __builtin_amdgcn_readfirstlane(p0);
    const bool turn = a.rope_cos;
    f32x4 x[2][2], cs[2], sn[2];
    unsigned was[2][2];
    bool adds[2], has[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = p0 + 16 * i, from = first + 16 * i;
      adds[i] = max(old, from) < min(end, from + ROWS);
      has[i] = old > from;
      if (has[i])
#pragma unroll
        for (int h = 0; h < 2; ++h) was[i][h] = *(const unsigned*)(dst + paged_k_offset(p, d + h * MID, HD));
      if (!adds[i]) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) x[i][h] = *(const f32x4*)(row(p) + d + h * MID);
      if (turn) {
        const size_t t = (size_t)(block * kBlk + near(p)) * MID + d;
        cs[i] = *(const f32x4*)(a.rope_cos + t);
        sn[i] = *(const f32x4*)(a.rope_sin + t);
      }
    }
    double y[2][2][4], amax = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!adds[i]) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        double u = x[i][0][k], w = x[i][1][k];
        if (turn) {
          const double c = cs[i][k], s = sn[i][k], u0 = u;
          u = u0 * c - w * s;
          w = u0 * s + w * c;
        }
        y[i][0][k] = u;
        y[i][1][k] = w;
        amax = fmax(amax, fmax(fabs(u), fabs(w)));  // passes over NaN
      }
    }
    e = max(e_old, exponent(amax));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = p0 + 16 * i;
      if (!adds[i] && !(has[i] && e > e_old)) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unsigned w = 0;
        if (adds[i])
#pragma unroll
          for (int k = 0; k < 4; ++k) w |= ((unsigned)code_of(y[i][h][k], e) & 255u) << (8 * k);
        if (p < old) w = e > e_old ? shift_word(was[i][h], min(e - e_old, 8), 0) : was[i][h];
        if (p < end) *(unsigned*)(dst + paged_k_offset(p, d + h * MID, HD)) = w;
      }
    }
  }
  if (tid == 0) a.pool.exps[unit] = (int8_t)e;
}
extern "C" __global__ __launch_bounds__(block_threads(64)) void paged_append_hd64(PagedRowsArgs a) { append_block<64>(a); }
extern "C" __global__ __launch_bounds__(block_threads(128)) void paged_append_hd128(PagedRowsArgs a) { append_block<128>(a); }

// Reads one block's rows of a range back as f32; a thread has the codes of the append.
// Bound by memory: 4 x 2048 rows of 8 heads x 128 in 18.3 us (median of 125 launches; the
// fastest 16.2), 84 MB at 4.6 to 5.2 TB/s.
template <int HD>
__device__ __forceinline__ void read_block(const PagedRowsArgs& a) {
  constexpr int MID = HD / 2, BYTES = kBlk * HD, LANES = MID / 4;
  const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
  const Seq q = find_seq(a.seqs, blockIdx.x);
  const int block = q.pos / kBlk + q.item;
  const int first = max(0, q.pos - block * kBlk), end = min(kBlk, q.pos + q.rows - block * kBlk);
  const size_t unit = ((size_t)pool_block(a.pool, q.slot, block) * a.pool.nkv + head) * 2 + which;
  const uint8_t* src = a.pool.codes + unit * BYTES;
  const float step = ldexpf(1.0f, a.pool.exps[unit]);
  float* dst = a.rows[which] + (size_t)head * HD;
  auto row = [&](int p) { return dst + (ptrdiff_t)(q.row0 + block * kBlk - q.pos + p) * (a.pool.nkv * HD); };
  if (which) {
    const int d = tid % HD, p0 = tid / HD * 16;
    if (max(first, p0) >= min(end, p0 + 16)) return;
    const u32x4 w = *(const u32x4*)(src + paged_v_offset(p0, d));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (p0 + i >= first && p0 + i < end)
        row(p0 + i)[d] = (float)((int)((w[i / 4] >> (8 * (i % 4))) & 255u) - 128) * step;
  } else {
    const int d = 4 * (tid % LANES), p0 = tid / LANES;
    unsigned w[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[i][h] = *(const unsigned*)(src + paged_k_offset(p0 + 16 * i, d + h * MID, HD));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = p0 + 16 * i;
      if (p < first || p >= end) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (float)((int)(w[i][h] << (24 - 8 * k)) >> 24) * step;
        *(f32x4*)(row(p) + d + h * MID) = x;
      }
    }
  }
}
extern "C" __global__ __launch_bounds__(block_threads(64)) void paged_read_hd64(PagedRowsArgs a) { read_block<64>(a); }
extern "C" __global__ __launch_bounds__(block_threads(128)) void paged_read_hd128(PagedRowsArgs a) { read_block<128>(a); }

// Attention of new rows over the cached positions.  A column is one (row, query
// head of the KV head's group); a wave takes 16 of them per group, and tiles of 64
// positions:
//   S^T = K Q^T    v_mfma_i32_16x16x64_i8: the K codes are the operand as they
//                  lie in the cache; q is a fixed-point number of 22 bits below
//                  its largest magnitude, in three signed bytes, so the sums are
//                  exact; a score is off by the rounding of q (2^-23 of its
//                  largest value), by less than a step of 2^-14 of it and the
//                  block's (the lowest byte's sum is rounded down, so always to one
//                  side), and by two f32 roundings.
//   softmax        online per column, exp2 of log2(e)-scaled scores.
//   O^T += V^T P^T v_mfma_f32_16x16x32_f16: the V codes as f16 (a byte placed in
//                  1024 + code + 128, less 1152), p times the block's scale as f16
//                  hi + lo.  The scales enter through the exponent: each column keeps the
//                  running maximum of score + e besides that of the score, and its
//                  weights are 2^(score + e - that) <= 1, whatever the sizes of V.
// Lane l of a tile: column c = l % 16, positions 16 (l / 16) .. + 15, all in one
// block, so both exponents are a lane's own.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3e38f;

// One value of q in fixed point: n = n2 2^16 + n1 2^8 + n0, three signed bytes, byte
// `b` of a word each.
__device__ __forceinline__ void put_bytes(float x, int ex, int b, unsigned (&w)[3]) {
  const int n = (int)rintf(ldexpf(x, ex));
  const int n1 = (n + 128) >> 8, n2 = (n1 + 128) >> 8;
  w[0] |= ((unsigned)n & 255u) << (8 * b);
  w[1] |= ((unsigned)n1 & 255u) << (8 * b);
  w[2] |= ((unsigned)n2 & 255u) << (8 * b);
}
// The exponent that takes a row's largest magnitude to [2^21, 2^22); rows that are
// not finite become zeros with a scale of NaN, so that only their column is NaN.
__device__ __forceinline__ int row_exp(float amax, bool odd) {
  return amax > 0.0f && !odd ? 22 - __builtin_amdgcn_frexp_expf(amax) : 0;
}
__device__ __forceinline__ float row_scale(float scale, int ex, bool odd) {
  return odd ? NAN : ldexpf(scale * kLog2e, 8 - ex);  // scores come in steps of 2^8
}

// Eight codes of V (positions of one half of a lane's 16) as f16.
__device__ __forceinline__ h16x8 v_half(unsigned w0, unsigned w1) {
  const h16x2 less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  h16x8 v;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned w = k ? w1 : w0;
    const h16x2 x = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + less;
    const h16x2 y = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + less;
    v[4 * k] = x.x;
    v[4 * k + 1] = x.y;
    v[4 * k + 2] = y.x;
    v[4 * k + 3] = y.y;
  }
  return v;
}

// What two weights have over their f16 parts, rounded to f16: the mixed-precision
// operation takes the f16 as it is (exact: hi * -1 + w).
__device__ __forceinline__ h16x2 rest(h16x2 hi, float w0, float w1) {
  const unsigned h = __builtin_bit_cast(unsigned, hi);
  float a, b;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(h), "v"(w0));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(h), "v"(w1));
  return h16x2{(_Float16)a, (_Float16)b};
}

// The maximum over the lanes that share l % 16.
__device__ __forceinline__ float group_max(float x) {
  auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// The running state of a wave's 16 columns.
template <int HD>
struct Column {
  // m: the largest score, far below every one and finite before the column has seen a
  // position, so that differences are numbers; g: how far the largest score + e lies
  // above m (a number of its own: next to a large score e would be lost)
  float m = kNone, g = 0.0f, l = 0.0f;  // l: of this lane's positions
  float oc = 1.0f;
  f32x4 o[HD / 16];                               // 2^(14 - m - g) O: dims 16 d + 4 r + i
  __device__ __forceinline__ Column() {
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Scores of a tile (not yet scaled) from the integer sums: the lowest bytes' sum
  // enters in whole steps of 2^8, rounded down like every other's, as what the next
  // bytes' sum starts from.
  template <int BH, class K, class Q>
  static __device__ __forceinline__ void scores(K&& k, Q&& q, float (&sv)[16]) {
    // BH operand rows at a time: their chains are independent of each other
#pragma unroll
    for (int b0 = 0; b0 < 4; b0 += BH) {
      i32x4 hi[BH], lo[BH];
#pragma unroll
      for (int b = 0; b < BH; ++b) lo[b] = hi[b] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < HD / 64; ++s)
#pragma unroll
        for (int b = 0; b < BH; ++b) lo[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k(b0 + b, s), q(0, s), lo[b], 0, 0, 0);
#pragma unroll
      for (int s = 0; s < HD / 64; ++s)
#pragma unroll
        for (int b = 0; b < BH; ++b) hi[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k(b0 + b, s), q(2, s), hi[b], 0, 0, 0);
#pragma unroll
      for (int b = 0; b < BH; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[b][i] >>= 8;
#pragma unroll
      for (int s = 0; s < HD / 64; ++s)
#pragma unroll
        for (int b = 0; b < BH; ++b) lo[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k(b0 + b, s), q(1, s), lo[b], 0, 0, 0);
#pragma unroll
      for (int b = 0; b < BH; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[4 * (b0 + b) + i] = (float)((hi[b][i] << 8) + lo[b][i]);
    }
  }

  // Positions that the column does not see: e > past.
  static __device__ __forceinline__ void hide(int past, float (&sv)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sv[e] = e > past ? -INFINITY : sv[e];
  }

  // Weights of a tile as f16 hi + lo; the state moves to the new maxima.
  __device__ __forceinline__ void weigh(const float (&sv)[16], float sl2, int ek, float ev, h16x8 (&ph)[2], h16x8 (&pl)[2]) {
    float mx = sv[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sv[e]);
    // the scale of q and the block: kept above zero, so that a position out of
    // sight stays at -inf (NaN is kept)
    float f = ldexpf(sl2, ek);
    f = f < 1e-38f ? 1e-38f : f;
    mx = mx * f;
    const float mn = fmaxf(m, group_max(mx)), up = g + (m - mn), gn = fmaxf(up, group_max(ev + (mx - mn)));
    // a weight is p 2^gain: 2^14 puts hi and lo in f16's range, and below 2^-30 both are
    // zero whatever the gain, while p still counts in the sum
    const float gain = fmaxf(ev - gn + 14.0f, -30.0f), less = gain - mn;
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __builtin_fmaf(sv[e], f, less);
    // where the last place of the maximum counts, scores are rounded as it is
    const bool coarse = fabsf(mn) > 0x1p20f && mn != kNone;
    if (__ballot(coarse))
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = coarse ? (sv[e] * f - mn) + gain : x[e];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float w0 = __builtin_amdgcn_exp2f(x[e]);
      const float w1 = __builtin_amdgcn_exp2f(x[e + 1]);
      sum += w0;
      sum += w1;
      const h16x2 hi = __builtin_bit_cast(h16x2, __builtin_amdgcn_cvt_pkrtz(w0, w1));
      const h16x2 lo = rest(hi, w0, w1);
      ph[e >> 3][e & 7] = hi.x;
      ph[e >> 3][(e & 7) + 1] = hi.y;
      pl[e >> 3][e & 7] = lo.x;
      pl[e >> 3][(e & 7) + 1] = lo.y;
    }
    l = l * __builtin_amdgcn_exp2f(m - mn) + sum * __builtin_amdgcn_exp2f(-gain);
    m = mn;
    oc = __builtin_amdgcn_exp2f(up - gn);
    g = gn;
  }
  // O to the new maximum, where a column's has risen.
  __device__ __forceinline__ void rescale() {
    if (__ballot(oc != 1.0f)) {
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d] = o[d] * oc;
    }
  }

  // The lanes' sums together, and O as the weighted mean of V.
  __device__ __forceinline__ void close() {
    l += xor16(l);
    l += xor32(l);
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(g - 14.0f) / l;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] = o[d] * f;
  }
};

// What a workgroup works on: a tile of `cols` columns and a split.
struct Item {
  Seq q;
  int item, head, n_rep, n_col, past, n_split, tile, split, from, to;
};
__device__ __forceinline__ Item item_of(const PagedAttnArgs& a, int cols, int unit) {
  Item t;
  const int nkv = a.pool.nkv;
  t.head = blockIdx.x % nkv;
  t.item = blockIdx.x / nkv;
  t.q = find_seq(a.seqs, t.item);
  t.n_rep = a.nq / nkv;
  t.n_col = t.q.rows * t.n_rep;
  t.past = t.q.pos - t.q.rows;
  t.n_split = (t.q.pos + a.chunk - 1) / a.chunk;
  t.tile = t.q.item / t.n_split;
  t.split = t.q.item % t.n_split;
  t.tile = (t.n_col + cols - 1) / cols - 1 - t.tile;  // the last rows see the most: they come first
  // up to the last position that any of the tile's columns sees
  const int chunk = ((t.q.pos + unit - 1) / unit + t.n_split - 1) / t.n_split * unit;  // splits of one length
  t.from = t.split * chunk;
  t.to = min(t.from + chunk, t.past + (min((t.tile + 1) * cols, t.n_col) - 1) / t.n_rep + 1);
  return t;
}
__device__ __forceinline__ float* out_row(const PagedAttnArgs& a, const Item& t, int col, int hd) {
  return a.out + ((size_t)(t.q.row0 + col / t.n_rep) * a.nq + t.head * t.n_rep + col % t.n_rep) * hd;
}
// Where the codes and the exponents of the two blocks of a tile start.
struct Place {
  size_t u0, u1;  // units of one block's K or V
};
__device__ __forceinline__ Place place_of(const PagedAttnArgs& a, const Item& t, int t0) {
  const int b = t0 / kBlk, nkv = a.pool.nkv;
  const int b0 = pool_block(a.pool, t.q.slot, b);
  const int b1 = pool_block(a.pool, t.q.slot, (b + 1) * kBlk < t.q.pos ? b + 1 : b);
  return {((size_t)b0 * nkv + t.head) * 2, ((size_t)b1 * nkv + t.head) * 2};
}

// A column's result in dims 16 d + 4 r .. of lane group r, or the split's part of it.
template <int HD>
__device__ __forceinline__ void put_dims(const PagedAttnArgs& a, const Item& t, int cols, int local, int d, f32x4 o) {
  const int r = lane_id() >> 4, col = t.tile * cols + local;
  if (col >= t.n_col) return;
  if (t.n_split == 1) {
    *(f32x4*)(out_row(a, t, col, HD) + 16 * d + 4 * r) = o;
  } else {
    const size_t unit = ((size_t)t.item * a.pool.nkv + t.head) * cols;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(dev_u32x4, o), dev_rsrc(a.part_o + unit * HD),
                                           (local * HD + 16 * d + 4 * r) * 4, 0, kSc1);
  }
}
// The maximum and sum of a split's column.
__device__ __forceinline__ void put_sum(const PagedAttnArgs& a, const Item& t, int cols, int local, float m, float l) {
  if (t.n_split == 1 || lane_id() >= 16 || t.tile * cols + local >= t.n_col) return;
  const size_t unit = ((size_t)t.item * a.pool.nkv + t.head) * cols;
  __builtin_amdgcn_raw_buffer_store_b64(dev_u32x2{__float_as_uint(m), __float_as_uint(l)}, dev_rsrc(a.part_ml + unit * 2), local * 8,
                                        0, kSc1);
}

// One wave joins the splits of U columns from `col` on (those past the tile's last are
// left out), reading up to B loads of each at once: lane s holds split s's (max, sum);
// the weighted rows then run over 16 bytes per lane, HD / 4 lanes a row.
template <int HD, int U, int B>
__device__ __forceinline__ void join_columns(const PagedAttnArgs& a, const Item& t, int cols, int col, int hop, const float* ml0,
                                             const float* src) {
  constexpr int LPR = HD / 4, SPL = LLMRS_WAVE / LPR;
  const int lane = lane_id(), ns = t.n_split, end = min(t.n_col - t.tile * cols, cols);
  float w[U];
  f32x4 acc[U];
  dev_u32x2 ml[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    ml[u] = __builtin_amdgcn_raw_buffer_load_b64(dev_rsrc(ml0), (min(lane, ns - 1) * hop + min(col + u, end - 1)) * 8, 0, kSc1);
  }
  for (int s0 = 0; s0 < ns; s0 += SPL * B) {
    dev_u32x4 x[U][B];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < B; ++k)
        x[u][k] = __builtin_amdgcn_raw_buffer_load_b128(
            dev_rsrc(src),
            ((min(s0 + k * SPL + lane / LPR, ns - 1) * hop + min(col + u, end - 1)) * HD + 4 * (lane % LPR)) * 4, 0, kSc1);
    if (s0 == 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float ms = lane < ns ? __uint_as_float(ml[u].x) : kNone;
        w[u] = __builtin_amdgcn_exp2f(ms - wave_max(ms)) * (lane < ns ? __uint_as_float(ml[u].y) : 0.0f);
        w[u] = w[u] / wave_sum(w[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < B; ++k) {  // splits past the last: weight 0 (their lanes hold none)
        const int s = s0 + k * SPL + lane / LPR;
        const float f = __shfl(w[u], s & 63);
        acc[u] = acc[u] + __builtin_bit_cast(f32x4, x[u][k]) * (s < ns ? f : 0.0f);
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (SPL == 4) acc[u][i] += xor16(acc[u][i]);
      acc[u][i] += xor32(acc[u][i]);
    }
    if (lane < LPR && col + u < end) *(f32x4*)(out_row(a, t, t.tile * cols + col + u, HD) + 4 * lane) = acc[u];
  }
}

// The tile's last workgroup (a ticket, no waiting) joins the splits, in split
// order: what it reads moved with device-scope stores, each waited for before the
// ticket was taken.  (Through one XCD's L2 instead, where a head's workgroups share
// one: 22.1 -> 21.7 us over 8 x 32768 positions, 30.4 -> 31.6 with 40 columns; not kept.)
// Its time is that of its rounds of loads, so a wave takes four columns at a time
// where a few splits leave it the registers, and else two.
template <int HD>
__device__ __forceinline__ void join_splits(const PagedAttnArgs& a, const Item& t, int cols, int* ticket) {
  if (t.n_split == 1) return;
  const int nkv = a.pool.nkv;
  const size_t first = (size_t)(t.item - t.split) * nkv + t.head;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  int* counter = a.tickets + first * kTicketStride;
  if (threadIdx.x == 0) *ticket = atomicAdd(counter, 1);
  __syncthreads();
  if (*ticket != t.n_split - 1) return;
  if (threadIdx.x == 0) dev_stu(counter, 0, 0u);  // as it was found, for the next launch
  const float* ml0 = a.part_ml + first * cols * 2;
  const float* src = a.part_o + first * cols * HD;
  const int end = min(t.n_col - t.tile * cols, cols), wave = __builtin_amdgcn_readfirstlane(wave_id());
  constexpr int SPL = 256 / HD;  // splits of a load
  if (t.n_split <= 2 * SPL) {
    for (int col = 4 * wave; col < end; col += 16) join_columns<HD, 4, 2>(a, t, cols, col, nkv * cols, ml0, src);
  } else {
    for (int col = 2 * wave; col < end; col += 8) join_columns<HD, 2, 8>(a, t, cols, col, nkv * cols, ml0, src);
  }
}

// 16 columns: the four waves take every fourth tile of the split each, with
// the codes straight from the cache, and merge through LDS.  q is prepared by all
// of them together, 16 lanes a column, while the first tile is on its way.
// Bound by the stream of codes where they are many: 64 sequences of 1000 to 4000
// positions, 331 MB, in 57 us (5.8 TB/s; a stream that only reads reaches 7.1); 8 heads
// of one sequence behind 32 k positions, 67 MB, in 18.4 us, of which the join of 32
// splits is about 4 (one CU reads their results at some 45 GB/s) and start and end 4.
// Short contexts are a chain of dependent accesses: 7.3 us for 512 positions.  32 and 48
// columns per workgroup read the cache less often and were slower at every size tried (16
// sequences, 5 rows of 4 heads behind 2100 positions: 22.8 us with 16, 27.5 and 48.4), as
// were three waves per SIMD (57 us became 60; registers spill).
template <int HD>
__device__ __forceinline__ void attend_few(const PagedAttnArgs& a) {
  constexpr int S = HD / 64, ND = HD / 16, MID = HD / 2, BYTES = kBlk * HD, WP = 4, COLS = 16, STEP = 64 * WP;
  __shared__ __align__(16) float so[WP * 16 * HD];
  __shared__ float sm[WP * COLS * 2];
  __shared__ __align__(16) i32x4 sq[3 * S * LLMRS_WAVE];
  __shared__ float ssl[COLS];
  __shared__ int ticket;
  const Item t = item_of(a, COLS, STEP);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int c = lane & 15, r = lane >> 4;
  const int col0 = t.tile * COLS;

  // K's registers take the next tile's codes once the scores are formed, V's once
  // the products are, so each load has half a tile's arithmetic to arrive in
  i32x4 kk[4][S];
  u32x4 vv[ND];
  unsigned exps = 0;  // of the lane's positions: K, V
  const uint8_t* vp = nullptr;
  auto fetch_k = [&](const Place& p) {
    const size_t uk = c < 8 ? p.u0 : p.u1, uv = r < 2 ? p.u0 : p.u1;
    exps = *(const uint16_t*)(a.pool.exps + uv);
    const uint8_t* kp = a.pool.codes + uk * BYTES + r * 128 + (c & 7) * 16;
    vp = a.pool.codes + (uv + 1) * BYTES + (r & 1) * 256 + c * 16;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int s = 0; s < S; ++s) kk[b][s] = __builtin_nontemporal_load((const i32x4*)(kp + (b * S + s) * 512));
  };
  auto fetch_v = [&] {
#pragma unroll
    for (int d = 0; d < ND; ++d) vv[d] = __builtin_nontemporal_load((const u32x4*)(vp + d * 512));
  };
  int t0 = t.from + 64 * wave;
  if (t0 < t.to) {
    fetch_k(place_of(a, t, t0));
    fetch_v();
  }
  __builtin_amdgcn_sched_barrier(0);
  {
    // column tid / 16, dims W j .. and their partners
    constexpr int W = MID / 16;
    const int j = tid & 15, col = min(col0 + (tid >> 4), t.n_col - 1);
    const float* x = a.q + ((size_t)(t.q.row0 + col / t.n_rep) * a.nq + t.head * t.n_rep + col % t.n_rep) * HD + W * j;
    float u[W], v[W], amax = 0.0f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      u[i] = x[i];
      v[i] = x[i + MID];
    }
    if (a.rope_cos) {
      const size_t at = (size_t)(t.past + col / t.n_rep) * MID + W * j;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float cs = a.rope_cos[at + i], sn = a.rope_sin[at + i], u0 = u[i];
        u[i] = u0 * cs - v[i] * sn;
        v[i] = u0 * sn + v[i] * cs;
      }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      amax = fmaxf(amax, fmaxf(fabsf(u[i]), fabsf(v[i])));
      fine = fine && fabsf(u[i]) < INFINITY && fabsf(v[i]) < INFINITY;
    }
    amax = max16(amax);
    const bool odd = max16(fine ? 0.0f : 1.0f) != 0.0f;
    const int ex = row_exp(amax, odd);
    unsigned wu[3] = {0, 0, 0}, wv[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      put_bytes(odd ? 0.0f : u[i], ex, i, wu);
      put_bytes(odd ? 0.0f : v[i], ex, i, wv);
    }
    // lane (column, dim group) of the operand: a run of 4 bytes per step with 128
    // dims, of 2 in each half of the 16 with 64
    const int at = ((j >> 2) * 16 + (tid >> 4)) * 16;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint8_t* dst = (uint8_t*)(sq + k * S * LLMRS_WAVE) + at;
      if constexpr (HD == 128) {
        *(unsigned*)(dst + 4 * (j & 3)) = wu[k];
        *(unsigned*)(dst + 1024 + 4 * (j & 3)) = wv[k];
      } else {
        *(uint16_t*)(dst + 2 * (j & 3)) = (uint16_t)wu[k];
        *(uint16_t*)(dst + 8 + 2 * (j & 3)) = (uint16_t)wv[k];
      }
    }
    if (j == 0) ssl[tid >> 4] = row_scale(a.scale, ex, odd);
  }
  // a barrier for LDS alone: __syncthreads would wait for the tile as well
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  const float sl2 = ssl[c];
  const int limit = t.past + min(col0 + c, t.n_col - 1) / t.n_rep;  // the column's last visible position
  const int lowest = t.past + col0 / t.n_rep;
  Column<HD> x;
  for (; t0 < t.to; t0 += STEP) {
    const int ek = (int8_t)(exps & 255);
    const float ev = (float)(int8_t)(exps >> 8);
    const bool more = t0 + STEP < t.to;
    const Place next = place_of(a, t, more ? t0 + STEP : t0);
    float sv[16];
    asm volatile("" ::: "memory");  // q is read again for every tile: its registers are worth more
    Column<HD>::template scores<4>([&](int b, int s) { return kk[b][s]; },
                                    [&](int k, int s) { return sq[(k * S + s) * LLMRS_WAVE + lane]; }, sv);
    if (t0 + 63 > lowest) Column<HD>::hide(limit - t0 - 16 * r, sv);
    __builtin_amdgcn_sched_barrier(0);
    if (more) fetch_k(next);
    __builtin_amdgcn_sched_barrier(0);
    h16x8 ph[2], pl[2];
    x.weigh(sv, sl2, ek, ev, ph, pl);
    x.rescale();
    // two dim blocks at a time: their products are independent of each other
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += 2) {
      h16x8 va[2][2];
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h) va[d][h] = v_half(vv[d0 + d][2 * h], vv[d0 + d][2 * h + 1]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 0; d < 2; ++d)
          x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d][h], ph[h], x.o[d0 + d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 2; ++d)
          x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d][h], pl[h], x.o[d0 + d], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) fetch_v();
    __builtin_amdgcn_sched_barrier(0);
  }
  // the waves' results, in order; each wave adds them in dims of its own
  x.close();
#pragma unroll
  for (int d = 0; d < ND; ++d) *(f32x4*)(so + (wave * 16 + c) * HD + 16 * d + 4 * r) = x.o[d];
  if (r == 0) {
    sm[(wave * 16 + c) * 2] = x.m;
    sm[(wave * 16 + c) * 2 + 1] = x.l;
  }
  __syncthreads();
  float M = sm[c * 2], L = 0.0f, cw[WP];
#pragma unroll
  for (int w = 1; w < WP; ++w) M = fmaxf(M, sm[(w * 16 + c) * 2]);
#pragma unroll
  for (int w = 0; w < WP; ++w) {
    cw[w] = __builtin_amdgcn_exp2f(sm[(w * 16 + c) * 2] - M) * sm[(w * 16 + c) * 2 + 1];
    L += cw[w];
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  for (int d = wave; d < ND; d += WP) {
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WP; ++w) acc = acc + *(const f32x4*)(so + (w * 16 + c) * HD + 16 * d + 4 * r) * (cw[w] * inv);
    put_dims<HD>(a, t, COLS, c, d, acc);
  }
  if (wave == 0) put_sum(a, t, COLS, c, M, L);
  join_splits<HD>(a, t, COLS, &ticket);
}

// More columns: each wave has 16 of its own and takes every tile of the split.  The
// workgroup brings a tile into LDS once, V already as f16, while the one before is
// computed.
// Bound by issue: a tile of 16 columns is 56 matrix instructions, 17 exp2 and about 220
// others, which in a loop of two or three waves per SIMD cost 8, 9.6 and 4.4 cycles of
// it: 1590 of the 2175 that a tile takes.  2048 rows of 32 heads behind 2048 positions
// are 187 to 199 us (the fastest and the median of 125 launches), 103 GFLOP of the formula.  No faster were 128 columns in eight waves,
// 32 columns per wave (346 us: registers spill; 64 dims: 150 against 136), the next tile's
// scores among this one's weights (205 to 215) and raised priority of the matrix
// instructions (208).
template <int HD>
__device__ __forceinline__ void attend_many(const PagedAttnArgs& a) {
  constexpr int S = HD / 64, ND = HD / 16, MID = HD / 2, BYTES = kBlk * HD, COLS = 64, T = kThreads;
  constexpr int KW = 4 * S * LLMRS_WAVE, VW = 2 * ND * LLMRS_WAVE;  // 16-byte words of a tile
  constexpr int PER = BYTES / 16;                                   // of a block's K or V codes
  constexpr int N = (2 * PER + T - 1) / T;                          // of them per thread and tile
  constexpr int DB = 2;                                             // dim blocks at a time
  __shared__ __align__(16) u32x4 sk[2][KW];
  __shared__ __align__(16) u32x4 sv16[2][VW];
  __shared__ int ticket;
  const Item t = item_of(a, COLS, 64);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int c = lane & 15, r = lane >> 4;
  const int col0 = t.tile * COLS + wave * 16;

  // word w of a tile: word w % PER of its block w / PER
  u32x4 gk[N], gv[N];
  auto fetch = [&](u32x4 (&g)[N], const Place& p, int v) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int w = tid + n * T;
      if (2 * PER % T == 0 || w < 2 * PER)
        g[n] = ((const u32x4*)(a.pool.codes + ((w < PER ? p.u0 : p.u1) + v) * BYTES))[w % PER];
    }
  };
  auto stage_k = [&](int buf) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int w = tid + n * T, j = w / PER, i = w % PER;
      if (2 * PER % T == 0 || w < 2 * PER) sk[buf][(i >> 3) * 16 + j * 8 + (i & 7)] = gk[n];
    }
  };
  auto stage_v = [&](int buf) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      // word (d, r2, c): positions 16 (2 j + r2) .. of dim 16 d + c
      const int w = tid + n * T, j = w / PER, i = w % PER;
      const int d = i >> 5, at = (2 * j + ((i >> 4) & 1)) * 16 + (i & 15);
      if (2 * PER % T == 0 || w < 2 * PER)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          sv16[buf][(d * 2 + h) * LLMRS_WAVE + at] = __builtin_bit_cast(u32x4, v_half(gv[n][2 * h], gv[n][2 * h + 1]));
    }
  };
  auto exps_of = [&](const Place& p) { return *(const uint16_t*)(a.pool.exps + (r < 2 ? p.u0 : p.u1)); };
  const int n_tile = max(t.to - t.from + 63, 0) / 64;
  unsigned exps = 0, exps_next = 0;
  auto fetch_tile = [&](int t0) {
    const Place p = place_of(a, t, t0);
    exps_next = exps_of(p);
    fetch(gk, p, 0);
    fetch(gv, p, 1);
  };
  if (n_tile) fetch_tile(t.from);
  __builtin_amdgcn_sched_barrier(0);

  i32x4 qb[3][S];
  float sl2;
  const int col = min(col0 + c, t.n_col - 1), limit = t.past + col / t.n_rep;  // the column's last visible position
  {
    const float* x = a.q + ((size_t)(t.q.row0 + col / t.n_rep) * a.nq + t.head * t.n_rep + col % t.n_rep) * HD;
    float v[S][16];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 w = *(const f32x4*)(x + (HD == 128 ? 64 * s + 16 * r + e : (e & 7) + 8 * r + (e >> 3) * 32));
        v[s][e] = w.x; v[s][e + 1] = w.y; v[s][e + 2] = w.z; v[s][e + 3] = w.w;
      }
    if (a.rope_cos) {
      const size_t at = (size_t)limit * MID + (HD == 128 ? 16 : 8) * r;
#pragma unroll
      for (int e = 0; e < (HD == 128 ? 16 : 8); ++e) {
        const float cs = a.rope_cos[at + e], sn = a.rope_sin[at + e];
        float &u = v[0][e], &w = HD == 128 ? v[S - 1][e] : v[0][(e + 8) & 15];
        const float u0 = u, w0 = w;
        u = u0 * cs - w0 * sn;
        w = u0 * sn + w0 * cs;
      }
    }
    float amax = 0.0f;
    bool fine = true;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        amax = fmaxf(amax, fabsf(v[s][e]));
        fine = fine && fabsf(v[s][e]) < INFINITY;
      }
    float bad = fine ? 0.0f : 1.0f;
    amax = fmaxf(amax, xor16(amax));
    amax = fmaxf(amax, xor32(amax));
    bad = fmaxf(bad, xor16(bad));
    const bool odd = fmaxf(bad, xor32(bad)) != 0.0f;
    const int ex = row_exp(amax, odd);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned w[3] = {0, 0, 0};
#pragma unroll
        for (int b = 0; b < 4; ++b) put_bytes(odd ? 0.0f : v[s][4 * k + b], ex, b, w);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
          asm("" : "+v"(w[n]));  // words: else the loop puts them together again for every tile
          qb[n][s][k] = (int)w[n];
        }
      }
    sl2 = row_scale(a.scale, ex, odd);
  }
  // the wave's own range: tiles that all of its columns see, and the last that one
  // of them does
  const int lowest = t.past + min(col0, t.n_col - 1) / t.n_rep;
  const int last = col0 < t.n_col ? t.past + (min(col0 + 16, t.n_col) - 1) / t.n_rep : -1;
  Column<HD> x;
  exps = exps_next;
  if (n_tile) {
    stage_k(0);
    stage_v(0);
  }
  __syncthreads();
  for (int n = 0; n < n_tile; ++n) {
    const int t0 = t.from + 64 * n, buf = n & 1;
    fetch_tile(min(t0 + 64, t.from + 64 * (n_tile - 1)));  // after the last: that one again, not used
    __builtin_amdgcn_sched_barrier(0);
    if (t0 <= last) {
      float sv[16];
      Column<HD>::template scores<2>([&](int b, int s) { return __builtin_bit_cast(i32x4, sk[buf][(b * S + s) * LLMRS_WAVE + lane]); },
                                      [&](int k, int s) { return qb[k][s]; }, sv);
      if (t0 + 63 > lowest) Column<HD>::hide(limit - t0 - 16 * r, sv);
      h16x8 ph[2], pl[2];
      x.weigh(sv, sl2, (int8_t)(exps & 255), (float)(int8_t)(exps >> 8), ph, pl);
      x.rescale();
#pragma unroll
      for (int d0 = 0; d0 < ND; d0 += DB)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          h16x8 va[DB];
#pragma unroll
          for (int d = 0; d < DB; ++d) va[d] = __builtin_bit_cast(h16x8, sv16[buf][((d0 + d) * 2 + h) * LLMRS_WAVE + lane]);
#pragma unroll
          for (int d = 0; d < DB; ++d) x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d], ph[h], x.o[d0 + d], 0, 0, 0);
#pragma unroll
          for (int d = 0; d < DB; ++d) x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d], pl[h], x.o[d0 + d], 0, 0, 0);
        }
    }
    exps = exps_next;
    stage_k(buf ^ 1);
    stage_v(buf ^ 1);
    __syncthreads();
  }
  x.close();
#pragma unroll
  for (int d = 0; d < ND; ++d) put_dims<HD>(a, t, COLS, wave * 16 + c, d, x.o[d]);
  put_sum(a, t, COLS, wave * 16 + c, x.m, x.l);
  join_splits<HD>(a, t, COLS, &ticket);
}

#define LLMRS_PAGED_ATTN(KIND, HD, WAVES, BODY)                                                               \
  extern "C" __global__ __launch_bounds__(kThreads, WAVES) void paged_attn_##KIND##_hd##HD(PagedAttnArgs a) { BODY; }
LLMRS_PAGED_ATTN(few, 64, 3, attend_few<64>(a))
LLMRS_PAGED_ATTN(many, 64, 3, attend_many<64>(a))
LLMRS_PAGED_ATTN(few, 128, 2, attend_few<128>(a))
LLMRS_PAGED_ATTN(many, 128, 3, attend_many<128>(a))

// Words of the host into device memory (words.h).
extern "C" __global__ __launch_bounds__(kThreads) void paged_words(WordsArgs a) {
  for (int i = threadIdx.x; i < a.n; i += kThreads) a.dst[i] = a.w[i];
}
