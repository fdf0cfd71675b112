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
  Seq q;
  if (s.n == 1) {
    q.item = item;
    q.slot = s.w[1];
    q.row0 = s.w[2];
    q.rows = s.w[3];
    q.pos = s.w[4];
    return q;
  }
  int i = -1;
  for (int b = 0; b < s.n; b += LLMRS_WAVE) {
    const int l = b + lane_id();
    i += __popcll(__ballot(l < s.n && word(s, l < s.n ? l : 0) <= item));
  }
  i = __builtin_amdgcn_readfirstlane(i);
  const int at = s.n + 4 * i;
  q.item = item - word(s, i);
  q.slot = word(s, at);
  q.row0 = word(s, at + 1);
  q.rows = word(s, at + 2);
  q.pos = word(s, at + 3);
  return q;
}

// The pool block that holds block `b` of a slot.
__device__ __forceinline__ int pool_block(const PagedPool& p, int slot, int b) {
  return (p.table[(size_t)slot * p.stride + (b >> p.shift)] << p.shift) + (b & ((1 << p.shift) - 1));
}

// The smallest e in [kPagedExpMin, kPagedExpMax] with amax <= 127 * 2^e: amax =
// f * 2^x with f in [1/2, 1), and 127 = 127/128 * 2^7.
__device__ __forceinline__ int needed_exp(double amax) {
  const int e = __builtin_amdgcn_frexp_exp(amax) - 7 + (__builtin_amdgcn_frexp_mant(amax) > 127.0 / 128.0 ? 1 : 0);
  return amax > 0.0 ? min(max(e, kPagedExpMin), kPagedExpMax) : kPagedExpMin;
}

// c * 2^-d to the nearest integer, half to even, for 0 <= d <= 8.
__device__ __forceinline__ int shift_code(int c, int d) {
  return d ? (c + ((1 << (d - 1)) - 1) + ((c >> d) & 1)) >> d : c;
}

// Largest magnitude the format holds; NaN counts as zero.
__device__ __forceinline__ double storable(double x) {
  constexpr double top = 127.0 * 2658455991569831745807614120560689152.0;  // 127 * 2^121
  return x != x ? 0.0 : fmin(fmax(x, -top), top);
}

}  // namespace

// Appends rows to one block of one sequence.  The block's codes pass through LDS:
// the older rows' are loaded and, where the new rows raise the exponent, rounded
// to the new step.  K is rotated in 64 bits (the products of f32 values are exact
// there), so a code does not depend on how a sum was rounded.
template <int HD>
__device__ __forceinline__ void append_block(const PagedRowsArgs& a) {
  constexpr int MID = HD / 2, BYTES = kBlk * HD, ROWS = kBlk / (kThreads / MID);  // rows per thread
  __shared__ __align__(16) uint8_t codes[BYTES];
  __shared__ double red[kThreads / LLMRS_WAVE];
  const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
  const Seq q = find_seq(a.seqs, blockIdx.x);
  const int block = q.pos / kBlk + q.item;                  // of the sequence
  const int old = max(0, q.pos - block * kBlk);             // rows already there
  const int end = min(kBlk, q.pos + q.rows - block * kBlk); // rows after
  const int pb = pool_block(a.pool, q.slot, block);
  const size_t unit = ((size_t)pb * a.pool.nkv + head) * 2 + which;
  uint8_t* dst = a.pool.codes + unit * BYTES;

  // this thread's values: rows old + g, old + g + G, ..., dims j and j + HD/2
  constexpr int G = kThreads / MID;
  const int j = tid % MID, g = tid / MID;
  const int row0 = q.row0 + block * kBlk - q.pos, width = a.pool.nkv * HD;  // row of the block's position 0
  const float* src = a.rows[which] + (size_t)head * HD + j;
  const bool turn = which == 0 && a.rope_cos;
  double lo[ROWS], hi[ROWS], amax = 0.0;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int p = i * G + g;
    lo[i] = hi[i] = 0.0;
    if (p >= old && p < end) {
      const float* x = src + (size_t)(row0 + p) * width;
      double u = x[0], w = x[MID];
      if (turn) {
        const size_t t = (size_t)(block * kBlk + p) * MID + j;
        const double c = a.rope_cos[t], s = a.rope_sin[t], u0 = u;
        u = u0 * c - w * s;
        w = u0 * s + w * c;
      }
      lo[i] = storable(u);
      hi[i] = storable(w);
      amax = fmax(amax, fmax(fabs(lo[i]), fabs(hi[i])));
    }
  }
  u32x4 was[BYTES / (16 * kThreads) ? BYTES / (16 * kThreads) : 1];
  constexpr int VECS = BYTES / 16;
  if (old)
    for (int i = tid, n = 0; i < VECS; i += kThreads, ++n) was[n] = ((const u32x4*)dst)[i];
  const int e_old = old ? a.pool.exps[unit] : kPagedExpMin;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) amax = fmax(amax, __shfl_xor(amax, o));
  if (lane_id() == 0) red[wave_id()] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / LLMRS_WAVE; ++w) amax = fmax(amax, red[w]);
  const int e = max(e_old, needed_exp(amax));
  const int bias = which ? 128 : 0;
  if (old) {
    const int d = min(e - e_old, 8);
    for (int i = tid, n = 0; i < VECS; i += kThreads, ++n) {
      u32x4 v = was[n];
      if (d) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          unsigned out = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int c = (int)(int8_t)((v[k] >> (8 * b)) ^ (which ? 0x80u : 0u));
            out |= ((unsigned)(shift_code(c, d) + bias) & 255u) << (8 * b);
          }
          v[k] = out;
        }
      }
      ((u32x4*)codes)[i] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int p = i * G + g;
    if (p >= old && p < end) {
      const int cl = (int)rint(ldexp(lo[i], -e)), ch = (int)rint(ldexp(hi[i], -e));
      codes[which ? paged_v_offset(p, j) : paged_k_offset(p, j, HD)] = (uint8_t)(cl + bias);
      codes[which ? paged_v_offset(p, j + MID) : paged_k_offset(p, j + MID, HD)] = (uint8_t)(ch + bias);
    }
  }
  __syncthreads();
  for (int i = tid; i < VECS; i += kThreads) ((u32x4*)dst)[i] = ((const u32x4*)codes)[i];
  if (tid == 0) a.pool.exps[unit] = (int8_t)e;
}
extern "C" __global__ __launch_bounds__(kThreads) void paged_append_hd64(PagedRowsArgs a) { append_block<64>(a); }
extern "C" __global__ __launch_bounds__(kThreads) void paged_append_hd128(PagedRowsArgs a) { append_block<128>(a); }

// Reads one block's rows of a range back as f32.
template <int HD>
__device__ __forceinline__ void read_block(const PagedRowsArgs& a) {
  constexpr int BYTES = kBlk * HD;
  __shared__ __align__(16) uint8_t codes[BYTES];
  const int tid = threadIdx.x, head = blockIdx.y, which = blockIdx.z;
  const Seq q = find_seq(a.seqs, blockIdx.x);
  const int block = q.pos / kBlk + q.item;
  const int first = max(0, q.pos - block * kBlk), end = min(kBlk, q.pos + q.rows - block * kBlk);
  const size_t unit = ((size_t)pool_block(a.pool, q.slot, block) * a.pool.nkv + head) * 2 + which;
  const u32x4* src = (const u32x4*)(a.pool.codes + unit * BYTES);
  for (int i = tid; i < BYTES / 16; i += kThreads) ((u32x4*)codes)[i] = src[i];
  const float step = ldexpf(1.0f, a.pool.exps[unit]);
  __syncthreads();
  const int row0 = q.row0 + block * kBlk - q.pos, width = a.pool.nkv * HD;
  float* dst = a.rows[which] + (size_t)head * HD;
  for (int i = tid; i < BYTES; i += kThreads) {
    const int p = i / HD, d = i % HD;
    if (p < first || p >= end) continue;
    const int c = which ? (int)codes[paged_v_offset(p, d)] - 128 : (int)(int8_t)codes[paged_k_offset(p, d, HD)];
    dst[(size_t)(row0 + p) * width + d] = (float)c * step;
  }
}
extern "C" __global__ __launch_bounds__(kThreads) void paged_read_hd64(PagedRowsArgs a) { read_block<64>(a); }
extern "C" __global__ __launch_bounds__(kThreads) void paged_read_hd128(PagedRowsArgs a) { read_block<128>(a); }

// Attention of new rows over the cached positions.  A column is one (row, query
// head of the KV head's group); a wave takes 16 of them per group, and tiles of 64
// positions:
//   S^T = K Q^T    v_mfma_i32_16x16x64_i8: the K codes are the operand as they
//                  lie in the cache; q is a fixed-point number of 22 bits below
//                  its largest magnitude, in three signed bytes, so the sums are
//                  exact and a score is off by the rounding of q (2^-23 of its
//                  largest value) and of two f32 operations.
//   softmax        online per column, exp2 of log2(e)-scaled scores.
//   O^T += V^T P^T v_mfma_f32_16x16x32_f16: the V codes as f16 (a byte placed in
//                  1024 + code + 128, less 1152), p times the block's scale as f16
//                  hi + lo.  The scales enter through the exponent: each column keeps the
//                  running maximum mw of score + e besides that of the score, and
//                  its weights are 2^(score + e - mw) <= 1, whatever the sizes of V.
// Lane l of a tile: column c = l % 16, positions 16 (l / 16) .. + 15, all in one
// block, so both exponents are a lane's own.
constexpr float kLog2e = 1.4426950408889634f;

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
  return odd ? NAN : ldexpf(scale * kLog2e, -ex);
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

// The running state of a wave's 16 columns.
template <int HD>
struct Column {
  float m = -INFINITY, mw = -INFINITY, l = 0.0f;  // l: of this lane's positions
  f32x4 o[HD / 16];                               // 2^(14 - mw) O: dims 16 d + 4 r + i
  __device__ __forceinline__ Column() {
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Scores of a tile (not yet scaled) from the integer sums, and their maximum.
  // past: the column's last visible position less the lane's first.
  template <class K, class Q>
  static __device__ __forceinline__ float scores(K&& k, Q&& q, bool cut, int past, float (&sv)[16]) {
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      i32x4 s2 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0}, s0 = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < HD / 64; ++s) {
        const i32x4 x = k(b, s);
        s2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, q(2, s), s2, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, q(1, s), s1, 0, 0, 0);
        s0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, q(0, s), s0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = __builtin_fmaf((float)((s2[i] << 8) + s1[i]), 256.0f, (float)s0[i]);
        if (cut && 4 * b + i > past) x = -INFINITY;
        sv[4 * b + i] = x;
        mx = fmaxf(mx, x);
      }
    }
    return mx;
  }

  // Weights of a tile as f16 hi + lo; the state moves to the new maxima.
  __device__ __forceinline__ void weigh(const float (&sv)[16], float mx, float sl2, int ek, float ev, h16x8 (&ph)[2],
                                        h16x8 (&pl)[2]) {
    // the scale of q and the block: kept above zero, so that a position out of
    // sight stays at -inf (NaN is kept)
    float f = ldexpf(sl2, ek);
    f = f < 1e-38f ? 1e-38f : f;
    mx = mx * f;
    float mb = mx + ev;
    mx = fmaxf(mx, xor16(mx));
    mb = fmaxf(mb, xor16(mb));
    mx = fmaxf(mx, xor32(mx));
    mb = fmaxf(mb, xor32(mb));
    const float mn = fmaxf(m, mx), wn = fmaxf(mw, mb);
    const float at = mn == -INFINITY ? 0.0f : mn;  // no position seen yet: every p is 2^-inf
    const float wt = wn == -INFINITY ? 0.0f : wn;
    l *= __builtin_amdgcn_exp2f(m - at);
    const float oc = __builtin_amdgcn_exp2f(mw - wt);
    // 2^14 puts the weights' hi and lo parts in f16's range
    const float gain = __builtin_amdgcn_exp2f(fminf(ev + at - wt, 100.0f) + 14.0f);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], f, -at));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e + 1], f, -at));
      sum += p0;
      sum += p1;
      float w0 = p0 * gain, w1 = p1 * gain;
      // hi has to be the rounded product's: unhindered, the compiler rounds
      // the exact one to f16 for the operand and this one for lo, an f16 step apart
      // where they fall on two sides of a tie
      asm("" : "+v"(w0), "+v"(w1));
      const h16x2 hi = __builtin_bit_cast(h16x2, __builtin_amdgcn_cvt_pkrtz(w0, w1));
      ph[e >> 3][e & 7] = hi.x;
      ph[e >> 3][(e & 7) + 1] = hi.y;
      pl[e >> 3][e & 7] = (_Float16)(w0 - (float)hi.x);
      pl[e >> 3][(e & 7) + 1] = (_Float16)(w1 - (float)hi.y);
    }
    l += sum;
    if (__ballot(wn != mw)) {
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d] = o[d] * oc;
    }
    m = mn;
    mw = wn;
  }

  // The lanes' sums together, and O as the weighted mean of V.
  __device__ __forceinline__ void close() {
    l += xor16(l);
    l += xor32(l);
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mw - m - 14.0f) / l;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] = o[d] * f;
  }
};

// What a workgroup works on: a tile of `cols` columns and a split.
struct Item {
  Seq q;
  int item, head, n_rep, n_col, past, n_split, tile, split, from, to;
};
__device__ __forceinline__ Item item_of(const PagedAttnArgs& a, int cols) {
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
  // up to the last position that any of the tile's columns sees
  t.from = t.split * a.chunk;
  t.to = min(t.from + a.chunk, t.past + (min((t.tile + 1) * cols, t.n_col) - 1) / t.n_rep + 1);
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
  const int b1 = (b + 1) * kBlk < t.q.pos ? pool_block(a.pool, t.q.slot, b + 1) : b0;
  return {((size_t)b0 * nkv + t.head) * 2, ((size_t)b1 * nkv + t.head) * 2};
}

// A column's result, or the split's part of it.
template <int HD>
__device__ __forceinline__ void put_column(const PagedAttnArgs& a, const Item& t, int cols, int local, const Column<HD>& x) {
  const int r = lane_id() >> 4, col = t.tile * cols + local;
  if (col >= t.n_col) return;
  if (t.n_split == 1) {
    float* dst = out_row(a, t, col, HD);
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) *(f32x4*)(dst + 16 * d + 4 * r) = x.o[d];
    return;
  }
  const size_t unit = ((size_t)t.item * a.pool.nkv + t.head) * cols;
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
    dev_st16(a.part_o + unit * HD, (local * HD + 16 * d + 4 * r) * 4, __builtin_bit_cast(dev_u32x4, x.o[d]));
  if (r == 0) {
    dev_stf(a.part_ml + unit * 2, local * 8, x.m);
    dev_stf(a.part_ml + unit * 2, local * 8 + 4, x.l);
  }
}

// The tile's last workgroup (a ticket, no waiting) joins the splits, in split
// order: what it reads moved with device-scope stores, each waited for before the
// ticket was taken.  A wave takes a column: lane s holds split s's (max, sum); the
// weighted rows then run over 16 bytes per lane, HD / 4 lanes a row.
template <int HD>
__device__ __forceinline__ void join_splits(const PagedAttnArgs& a, const Item& t, int cols, int* ticket) {
  if (t.n_split == 1) return;
  const int nkv = a.pool.nkv, lane = lane_id();
  const size_t first = (size_t)(t.item - t.split) * nkv + t.head;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) *ticket = atomicAdd(a.tickets + first * kTicketStride, 1);
  __syncthreads();
  if (*ticket != t.n_split - 1) return;
  if (threadIdx.x == 0) dev_stu(a.tickets + first * kTicketStride, 0, 0u);  // as it was found, for the next launch
  constexpr int LPR = HD / 4, SPL = LLMRS_WAVE / LPR, BATCH = 16;
  const float* ml0 = a.part_ml + first * cols * 2;
  const float* src = a.part_o + first * cols * HD;
  const int hop = nkv * cols, tile_cols = min(t.n_col - t.tile * cols, cols), ns = t.n_split;
  for (int col = __builtin_amdgcn_readfirstlane(wave_id()); col < tile_cols; col += kThreads / LLMRS_WAVE) {
    const dev_u32x2 ml = dev_ld8(ml0, (min(lane, ns - 1) * hop + col) * 8);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float w = 0.0f;
    for (int s0 = 0; s0 < ns; s0 += SPL * BATCH) {
      dev_u32x4 x[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (s0 + k * SPL < ns) x[k] = dev_ld16(src, ((min(s0 + k * SPL + lane / LPR, ns - 1) * hop + col) * HD + 4 * (lane % LPR)) * 4);
      if (s0 == 0) {
        const float ms = lane < ns ? __uint_as_float(ml.x) : -INFINITY;
        const float M = wave_max(ms);
        w = __builtin_amdgcn_exp2f(ms - (M == -INFINITY ? 0.0f : M)) * (lane < ns ? __uint_as_float(ml.y) : 0.0f);
        w = w / wave_sum(w);
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (s0 + k * SPL < ns) acc = acc + __builtin_bit_cast(f32x4, x[k]) * __shfl(w, min(s0 + k * SPL + lane / LPR, 63));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (SPL == 4) acc[i] += xor16(acc[i]);
      acc[i] += xor32(acc[i]);
    }
    if (lane < LPR) *(f32x4*)(out_row(a, t, t.tile * cols + col, HD) + 4 * lane) = acc;
  }
}

// Up to 16 columns: the four waves take every fourth tile of the split each, with
// the codes straight from the cache, and merge through LDS.  q is prepared by all
// of them together, 16 lanes a column, while the first tile is on its way.
template <int HD>
__device__ __forceinline__ void attend_few(const PagedAttnArgs& a) {
  constexpr int S = HD / 64, ND = HD / 16, MID = HD / 2, BYTES = kBlk * HD, WP = 4, COLS = 16, STEP = 64 * WP;
  __shared__ __align__(16) float so[WP * COLS * HD];
  __shared__ float sm[WP * COLS * 2];
  __shared__ __align__(16) i32x4 sq[3 * S * LLMRS_WAVE];
  __shared__ float ssl[COLS];
  __shared__ int ticket;
  const Item t = item_of(a, COLS);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int c = lane & 15, r = lane >> 4;
  const int col0 = t.tile * COLS;

  // K's registers take the next tile's codes once the scores are formed, V's once
  // the products are, so each load has half a tile's arithmetic to arrive in
  i32x4 kk[4][S];
  u32x4 vv[ND];
  unsigned exps = 0;  // of the lane's positions: K, V
  const uint8_t* vp = nullptr;
  auto fetch_k = [&](int t0) {
    const Place p = place_of(a, t, t0);
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
    fetch_k(t0);
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
      uint8_t* dst = (uint8_t*)sq + k * S * 1024 + at;
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
  __syncthreads();
  const float sl2 = ssl[c];
  const int limit = t.past + min(col0 + c, t.n_col - 1) / t.n_rep, lowest = t.past + col0 / t.n_rep;
  Column<HD> x;
  for (; t0 < t.to; t0 += STEP) {
    const int ek = (int8_t)(exps & 255);
    const float ev = (float)(int8_t)(exps >> 8);
    float sv[16];
    asm volatile("" ::: "memory");  // q is read again for every tile: its registers are worth more
    const float mx = Column<HD>::scores([&](int b, int s) { return kk[b][s]; },
                                        [&](int k, int s) { return sq[(k * S + s) * LLMRS_WAVE + lane]; }, t0 + 63 > lowest,
                                        limit - t0 - 16 * r, sv);
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + STEP < t.to) fetch_k(t0 + STEP);
    __builtin_amdgcn_sched_barrier(0);
    h16x8 ph[2], pl[2];
    x.weigh(sv, mx, sl2, ek, ev, ph, pl);
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
        for (int d = 0; d < 2; ++d) x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d][h], ph[h], x.o[d0 + d], 0, 0, 0);
#pragma unroll
        for (int d = 0; d < 2; ++d) x.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d][h], pl[h], x.o[d0 + d], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + STEP < t.to) fetch_v();
    __builtin_amdgcn_sched_barrier(0);
  }
  x.close();
#pragma unroll
  for (int d = 0; d < ND; ++d) *(f32x4*)(so + (wave * COLS + c) * HD + 16 * d + 4 * r) = x.o[d];
  if (r == 0) {
    sm[(wave * COLS + c) * 2] = x.m;
    sm[(wave * COLS + c) * 2 + 1] = x.l;
  }
  __syncthreads();
  if (wave == 0) {
    float M = x.m;
#pragma unroll
    for (int w = 1; w < WP; ++w) M = fmaxf(M, sm[(w * COLS + c) * 2]);
    const float at = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, cw[WP];
#pragma unroll
    for (int w = 0; w < WP; ++w) {
      cw[w] = __builtin_amdgcn_exp2f(sm[(w * COLS + c) * 2] - at) * sm[(w * COLS + c) * 2 + 1];
      L += cw[w];
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < WP; ++w) acc = acc + *(const f32x4*)(so + (w * COLS + c) * HD + 16 * d + 4 * r) * (cw[w] * inv);
      x.o[d] = acc;
    }
    x.m = M;
    x.l = L;
    put_column<HD>(a, t, COLS, c, x);
  }
  join_splits<HD>(a, t, COLS, &ticket);
}

// More columns: a wave has 16 NG of its own and takes every tile of the split.  The
// workgroup brings a tile into LDS once, V already as f16, while the one before is
// computed.
template <int HD, int NG>
__device__ __forceinline__ void attend_many(const PagedAttnArgs& a) {
  constexpr int S = HD / 64, ND = HD / 16, MID = HD / 2, BYTES = kBlk * HD, COLS = 64 * NG;
  constexpr int KW = 4 * S * LLMRS_WAVE, VW = 2 * ND * LLMRS_WAVE;  // 16-byte words of a tile
  constexpr int PER = BYTES / 16;                                   // of a block's K or V codes
  constexpr int N = 2 * PER / kThreads;                             // of them per thread and tile: 1 or 2
  __shared__ __align__(16) u32x4 sk[2][KW];
  __shared__ __align__(16) u32x4 sv16[2][VW];
  __shared__ int ticket;
  const Item t = item_of(a, COLS);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int c = lane & 15, r = lane >> 4;
  const int col0 = t.tile * COLS + wave * 16 * NG;

  // word w of block j of the tile
  u32x4 gk[N], gv[N];
  unsigned exps = 0, exps_next = 0;
  auto fetch = [&](int t0) {
    const Place p = place_of(a, t, t0);
    exps_next = *(const uint16_t*)(a.pool.exps + (r < 2 ? p.u0 : p.u1));
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int j = N == 2 ? n : tid / PER, w = N == 2 ? tid : tid % PER;
      const u32x4* src = (const u32x4*)(a.pool.codes + (j ? p.u1 : p.u0) * BYTES) + w;
      gk[n] = src[0];
      gv[n] = src[PER];
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int j = N == 2 ? n : tid / PER, w = N == 2 ? tid : tid % PER;
      sk[buf][(w >> 3) * 16 + j * 8 + (w & 7)] = gk[n];
      // V word (d, r2, c): positions 16 (2 j + r2) .. of dim 16 d + c
      const int d = w >> 5, at = (2 * j + ((w >> 4) & 1)) * 16 + (w & 15);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sv16[buf][(d * 2 + h) * LLMRS_WAVE + at] = __builtin_bit_cast(u32x4, v_half(gv[n][2 * h], gv[n][2 * h + 1]));
    }
  };
  if (t.from < t.to) fetch(t.from);
  __builtin_amdgcn_sched_barrier(0);

  i32x4 qb[NG][3][S];
  float sl2[NG];
  int limit[NG];  // the column's last visible position
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int col = min(col0 + 16 * g + c, t.n_col - 1);
    limit[g] = t.past + col / t.n_rep;
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
      const size_t at = (size_t)limit[g] * MID + (HD == 128 ? 16 : 8) * r;
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
        for (int n = 0; n < 3; ++n) qb[g][n][s][k] = (int)w[n];
      }
    sl2[g] = row_scale(a.scale, ex, odd);
  }
  // the wave's own range: from a tile that all of its columns see to the last that
  // one of them does
  const int lowest = t.past + min(col0, t.n_col - 1) / t.n_rep;
  const int last = col0 < t.n_col ? t.past + (min(col0 + 16 * NG, t.n_col) - 1) / t.n_rep : -1;
  Column<HD> x[NG];
  exps = exps_next;
  if (t.from < t.to) stage(0);
  __syncthreads();
  int buf = 0;
  for (int t0 = t.from; t0 < t.to; t0 += 64, buf ^= 1) {
    const bool more = t0 + 64 < t.to;
    if (more) fetch(t0 + 64);
    __builtin_amdgcn_sched_barrier(0);
    if (t0 <= last) {
      const int ek = (int8_t)(exps & 255);
      const float ev = (float)(int8_t)(exps >> 8);
      h16x8 ph[NG][2], pl[NG][2];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sv[16];
        const float mx = Column<HD>::scores(
            [&](int b, int s) { return __builtin_bit_cast(i32x4, sk[buf][(b * S + s) * LLMRS_WAVE + lane]); },
            [&](int k, int s) { return qb[g][k][s]; }, t0 + 63 > lowest, limit[g] - t0 - 16 * r, sv);
        x[g].weigh(sv, mx, sl2[g], ek, ev, ph[g], pl[g]);
      }
#pragma unroll
      for (int d0 = 0; d0 < ND; d0 += 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          h16x8 va[2];
#pragma unroll
          for (int d = 0; d < 2; ++d) va[d] = __builtin_bit_cast(h16x8, sv16[buf][((d0 + d) * 2 + h) * LLMRS_WAVE + lane]);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int d = 0; d < 2; ++d)
              x[g].o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d], ph[g][h], x[g].o[d0 + d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 2; ++d)
              x[g].o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[d], pl[g][h], x[g].o[d0 + d], 0, 0, 0);
          }
        }
    }
    exps = exps_next;
    if (more) stage(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    x[g].close();
    put_column<HD>(a, t, COLS, wave * 16 * NG + 16 * g + c, x[g]);
  }
  join_splits<HD>(a, t, COLS, &ticket);
}

extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd64_few(PagedAttnArgs a) { attend_few<64>(a); }
extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd128_few(PagedAttnArgs a) { attend_few<128>(a); }
extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd64_many1(PagedAttnArgs a) { attend_many<64, 1>(a); }
extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd128_many1(PagedAttnArgs a) { attend_many<128, 1>(a); }
extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd64_many2(PagedAttnArgs a) { attend_many<64, 2>(a); }
extern "C" __global__ __launch_bounds__(kThreads, 2) void paged_attn_hd128_many2(PagedAttnArgs a) { attend_many<128, 2>(a); }

// Words of the host into device memory (words.h).
extern "C" __global__ __launch_bounds__(kThreads) void paged_words(WordsArgs a) {
  for (int i = threadIdx.x; i < a.n; i += kThreads) a.dst[i] = a.w[i];
}
