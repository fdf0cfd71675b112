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
  int i = -1;
  for (int b = 0; b < s.n; b += LLMRS_WAVE) {
    const int l = b + lane_id();
    i += __popcll(__ballot(l < s.n && word(s, l < s.n ? l : 0) <= item));
  }
  i = __builtin_amdgcn_readfirstlane(i);
  const int at = s.n + 4 * i;
  Seq q;
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
// head of the KV head's group); a workgroup's four waves are WC column groups of
// 16 * NG columns times WP = 4 / WC position groups, each of which takes every
// WP-th tile of 64 positions of the split.
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
template <int HD, int WC, int NG>
struct AttnShape {
  static constexpr int S = HD / 64, ND = HD / 16, WP = 4 / WC, COLS = 16 * NG * WC;
  static constexpr int LDS = WP > 1 ? WP * 16 * NG * WC * (HD + 2) : 1;  // floats
};

template <int HD, int WC, int NG>
__device__ __forceinline__ void attend(const PagedAttnArgs& a, float* lds) {
  typedef AttnShape<HD, WC, NG> SH;
  constexpr int S = SH::S, ND = SH::ND, WP = SH::WP, COLS = SH::COLS, MID = HD / 2, BYTES = kBlk * HD;
  constexpr float kLog2e = 1.4426950408889634f;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int c = lane & 15, r = lane >> 4;
  const int wc = wave % WC, wp = wave / WC;
  const int nkv = a.pool.nkv, n_rep = a.nq / nkv;
  const int head = blockIdx.x % nkv, item = blockIdx.x / nkv;
  const Seq q = find_seq(a.seqs, item);
  const int n_split = (q.pos + a.chunk - 1) / a.chunk;
  const int tile = q.item / n_split, split = q.item % n_split;
  const int n_col = q.rows * n_rep, col0 = tile * COLS + wc * 16 * NG;
  const int past = q.pos - q.rows;

  // q: the column's row, rotated, in three signed bytes per value
  i32x4 qb[NG][3][S];
  float sl2[NG];
  int limit[NG];  // the column's last visible position
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int col = min(col0 + 16 * g + c, n_col - 1);
    const int t = col / n_rep, h = head * n_rep + col % n_rep;
    limit[g] = past + t;
    const float* x = a.q + ((size_t)(q.row0 + t) * a.nq + h) * HD;
    float v[S][16];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = HD == 128 ? 64 * s + 16 * r + e : (e & 7) + 8 * r + (e >> 3) * 32;
        const f32x4 w = *(const f32x4*)(x + d);
        v[s][e] = w.x; v[s][e + 1] = w.y; v[s][e + 2] = w.z; v[s][e + 3] = w.w;
      }
    if (a.rope_cos) {
      const size_t at = (size_t)limit[g] * MID + (HD == 128 ? 16 : 8) * r;
#pragma unroll
      for (int e = 0; e < (HD == 128 ? 16 : 8); ++e) {
        const float cs = a.rope_cos[at + e], sn = a.rope_sin[at + e];
        float &u = v[0][e], &w = HD == 128 ? v[S - 1][e] : v[0][e + 8 < 16 ? e + 8 : 0];
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
    float odd = fine ? 0.0f : 1.0f;  // a NaN or an infinity in the row: NaN for the column
    amax = fmaxf(amax, xor16(amax));
    amax = fmaxf(amax, xor32(amax));
    odd = fmaxf(odd, xor16(odd));
    odd = fmaxf(odd, xor32(odd));
    const int ex = amax > 0.0f && odd == 0.0f ? 22 - __builtin_amdgcn_frexp_expf(amax) : 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned b0 = 0, b1 = 0, b2 = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int n = odd != 0.0f ? 0 : (int)rintf(ldexpf(v[s][4 * k + b], ex));
          const int n1 = (n + 128) >> 8, n2 = (n1 + 128) >> 8;  // n = n2 2^16 + (n1 - 256 n2) 2^8 + (n - 256 n1)
          b0 |= ((unsigned)n & 255u) << (8 * b);
          b1 |= ((unsigned)n1 & 255u) << (8 * b);
          b2 |= ((unsigned)n2 & 255u) << (8 * b);
        }
        qb[g][0][s][k] = (int)b0;
        qb[g][1][s][k] = (int)b1;
        qb[g][2][s][k] = (int)b2;
      }
    sl2[g] = odd != 0.0f ? NAN : ldexpf(a.scale * kLog2e, -ex);
  }

  float m[NG], mw[NG], l[NG];
  f32x4 o[NG][ND];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    m[g] = mw[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[g][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // the split's tiles up to the last position that any of the wave's columns sees
  const int last = past + (min(col0 + 16 * NG, n_col) - 1) / n_rep, lowest = past + min(col0, n_col - 1) / n_rep;
  const int from = split * a.chunk, to = min(from + a.chunk, (col0 < n_col ? last : -1) + 1);
  const int n_block = (q.pos + kBlk - 1) / kBlk;
  for (int t0 = from + 64 * wp; t0 < to; t0 += 64 * WP) {
    const int bl = t0 / kBlk;
    const int pb0 = pool_block(a.pool, q.slot, bl), pb1 = bl + 1 < n_block ? pool_block(a.pool, q.slot, bl + 1) : pb0;
    const size_t u0 = ((size_t)pb0 * nkv + head) * 2, u1 = ((size_t)pb1 * nkv + head) * 2;
    const size_t uk = c < 8 ? u0 : u1, uv = r < 2 ? u0 : u1;
    const uint16_t ee = *(const uint16_t*)(a.pool.exps + uv);
    const float ek = (float)(int8_t)(ee & 255), ev = (float)(int8_t)(ee >> 8);
    const uint8_t* kp = a.pool.codes + uk * BYTES + r * 128 + (c & 7) * 16;
    const uint8_t* vp = a.pool.codes + (uv + 1) * BYTES + (r & 1) * 256 + c * 16;
    i32x4 kk[4][S];
    u32x4 vv[ND];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int s = 0; s < S; ++s) kk[b][s] = *(const i32x4*)(kp + (b * S + s) * 512);
#pragma unroll
    for (int d = 0; d < ND; ++d) vv[d] = *(const u32x4*)(vp + d * 512);

    h16x8 ph[NG][2], pl[NG][2];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sv[16];
      const float f = ldexpf(sl2[g], (int)ek);
      float mt = -INFINITY;
      const bool cut = t0 + 63 > lowest;  // some column does not see the whole tile
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        i32x4 s2 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0}, s0 = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) {
          s2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[b][s], qb[g][2][s], s2, 0, 0, 0);
          s1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[b][s], qb[g][1][s], s1, 0, 0, 0);
          s0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[b][s], qb[g][0][s], s0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = __builtin_fmaf((float)((s2[i] << 8) + s1[i]), 256.0f, (float)s0[i]) * f;
          if (cut && t0 + 16 * r + 4 * b + i > limit[g]) x = -INFINITY;
          sv[4 * b + i] = x;
          mt = fmaxf(mt, x);
        }
      }
      float mb = mt + ev;
      mt = fmaxf(mt, xor16(mt));
      mb = fmaxf(mb, xor16(mb));
      mt = fmaxf(mt, xor32(mt));
      mb = fmaxf(mb, xor32(mb));
      const float mn = fmaxf(m[g], mt), wn = fmaxf(mw[g], mb);
      const float at = mn == -INFINITY ? 0.0f : mn;  // no position seen yet: every p is 2^-inf
      const float wt = wn == -INFINITY ? 0.0f : wn;
      l[g] *= __builtin_amdgcn_exp2f(m[g] - at);
      const float oc = __builtin_amdgcn_exp2f(mw[g] - wt);
      // 2^14 puts the weights' hi and lo parts in f16's range
      const float gain = __builtin_amdgcn_exp2f(fminf(ev + at - wt, 100.0f) + 14.0f);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float p = __builtin_amdgcn_exp2f(sv[e] - at);
        sum += p;
        float w = p * gain;
        // hi has to be the rounded product's: unhindered, the compiler rounds
        // the exact one to f16 for the operand and this one for lo, an f16 step apart
        // where they fall on two sides of a tie
        asm("" : "+v"(w));
        const _Float16 hi = (_Float16)w;
        ph[g][e >> 3][e & 7] = hi;
        pl[g][e >> 3][e & 7] = (_Float16)(w - (float)hi);
      }
      l[g] += sum;  // this lane's positions; the groups are added after the loop
      if (__ballot(wn != mw[g])) {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[g][d] = o[g][d] * oc;
      }
      m[g] = mn;
      mw[g] = wn;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      h16x8 va[2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const h16x2 less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const h16x2 x = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, vv[d][k], 0x04010400u)) + less;
        const h16x2 y = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, vv[d][k], 0x04030402u)) + less;
        va[k >> 1][4 * (k & 1)] = x.x;
        va[k >> 1][4 * (k & 1) + 1] = x.y;
        va[k >> 1][4 * (k & 1) + 2] = y.x;
        va[k >> 1][4 * (k & 1) + 3] = y.y;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[0], ph[g][0], o[g][d], 0, 0, 0);
        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[1], ph[g][1], o[g][d], 0, 0, 0);
        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[0], pl[g][0], o[g][d], 0, 0, 0);
        o[g][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[1], pl[g][1], o[g][d], 0, 0, 0);
      }
    }
  }

  // (max, sum, O) of the wave's positions, O as a weighted mean
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    l[g] += xor16(l[g]);
    l[g] += xor32(l[g]);
    const float f = l[g] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mw[g] - m[g] - 14.0f) / l[g];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[g][d] = o[g][d] * f;
  }
  // the position groups' results, by group in order
  if constexpr (WP > 1) {
    float* so = lds;                                  // [wp][column][HD]
    float* sm = lds + WP * COLS * HD;                 // [wp][column][2]
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int col = wc * 16 * NG + 16 * g + c;
#pragma unroll
      for (int d = 0; d < ND; ++d) *(f32x4*)(so + ((size_t)wp * COLS + col) * HD + 16 * d + 4 * r) = o[g][d];
      if (r == 0) {
        sm[(wp * COLS + col) * 2] = m[g];
        sm[(wp * COLS + col) * 2 + 1] = l[g];
      }
    }
    __syncthreads();
    if (wp != 0) return;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int col = wc * 16 * NG + 16 * g + c;
      float M = m[g];
#pragma unroll
      for (int w = 1; w < WP; ++w) M = fmaxf(M, sm[(w * COLS + col) * 2]);
      const float at = M == -INFINITY ? 0.0f : M;
      float L = 0.0f, cw[WP];
#pragma unroll
      for (int w = 0; w < WP; ++w) {
        cw[w] = __builtin_amdgcn_exp2f(sm[(w * COLS + col) * 2] - at) * sm[(w * COLS + col) * 2 + 1];
        L += cw[w];
      }
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WP; ++w)
          acc = acc + *(const f32x4*)(so + ((size_t)w * COLS + col) * HD + 16 * d + 4 * r) * (cw[w] * inv);
        o[g][d] = acc;
      }
      m[g] = M;
      l[g] = L;
    }
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int local = wc * 16 * NG + 16 * g + c, col = tile * COLS + local;
    if (col >= n_col) continue;
    float* dst;
    if (n_split == 1) {
      dst = a.out + ((size_t)(q.row0 + col / n_rep) * a.nq + head * n_rep + col % n_rep) * HD;
    } else {
      const size_t at = ((size_t)item * nkv + head) * COLS + local;
      dst = a.part_o + at * HD;
      if (r == 0) {
        a.part_ml[2 * at] = m[g];
        a.part_ml[2 * at + 1] = l[g];
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) *(f32x4*)(dst + 16 * d + 4 * r) = o[g][d];
  }
}

// Joins the splits of a column tile: the workgroup of the tile's first item, a
// column per wave and round, in split order.
template <int HD>
__device__ __forceinline__ void join_splits(const PagedAttnArgs& a, int cols) {
  const int nkv = a.pool.nkv, n_rep = a.nq / nkv, lane = lane_id();
  const int head = blockIdx.x % nkv, item = blockIdx.x / nkv;
  const Seq q = find_seq(a.seqs, item);
  const int n_split = (q.pos + a.chunk - 1) / a.chunk;
  if (n_split == 1 || q.item % n_split) return;
  const int col0 = q.item / n_split * cols, n_col = min(q.rows * n_rep - col0, cols);
  const size_t step = (size_t)nkv * cols;
  for (int c = wave_id(); c < n_col; c += kThreads / LLMRS_WAVE) {
    const size_t at = ((size_t)item * nkv + head) * cols + c;
    float M = -INFINITY;
    for (int s = 0; s < n_split; ++s) M = fmaxf(M, a.part_ml[2 * (at + s * step)]);
    float L = 0.0f, acc[HD / 64];
#pragma unroll
    for (int d = 0; d < HD / 64; ++d) acc[d] = 0.0f;
    if (M == -INFINITY) M = 0.0f;
    for (int s = 0; s < n_split; ++s) {
      const float w = __builtin_amdgcn_exp2f(a.part_ml[2 * (at + s * step)] - M) * a.part_ml[2 * (at + s * step) + 1];
      L += w;
#pragma unroll
      for (int d = 0; d < HD / 64; ++d) acc[d] += w * a.part_o[(at + s * step) * HD + 64 * d + lane];
    }
    const int col = col0 + c;
    float* dst = a.out + ((size_t)(q.row0 + col / n_rep) * a.nq + head * n_rep + col % n_rep) * HD;
#pragma unroll
    for (int d = 0; d < HD / 64; ++d) dst[64 * d + lane] = acc[d] / L;
  }
}

#define LLMRS_PAGED_ATTN(HD, WC, NG)                                                              \
  extern "C" __global__ __launch_bounds__(kThreads) void paged_attn_hd##HD##_c##WC##g##NG(PagedAttnArgs a) { \
    __shared__ __align__(16) float lds[AttnShape<HD, WC, NG>::LDS];                               \
    attend<HD, WC, NG>(a, lds);                                                                   \
  }
LLMRS_PAGED_ATTN(64, 1, 1)
LLMRS_PAGED_ATTN(64, 1, 2)
LLMRS_PAGED_ATTN(64, 2, 2)
LLMRS_PAGED_ATTN(64, 4, 2)
LLMRS_PAGED_ATTN(128, 1, 1)
LLMRS_PAGED_ATTN(128, 1, 2)
LLMRS_PAGED_ATTN(128, 2, 2)
LLMRS_PAGED_ATTN(128, 4, 2)
#define LLMRS_PAGED_JOIN(HD, COLS) \
  extern "C" __global__ __launch_bounds__(kThreads) void paged_join_hd##HD##_##COLS(PagedAttnArgs a) { join_splits<HD>(a, COLS); }
LLMRS_PAGED_JOIN(64, 16)
LLMRS_PAGED_JOIN(64, 32)
LLMRS_PAGED_JOIN(64, 64)
LLMRS_PAGED_JOIN(64, 128)
LLMRS_PAGED_JOIN(128, 16)
LLMRS_PAGED_JOIN(128, 32)
LLMRS_PAGED_JOIN(128, 64)
LLMRS_PAGED_JOIN(128, 128)

// Words of the host into device memory (words.h).
extern "C" __global__ __launch_bounds__(kThreads) void paged_words(WordsArgs a) {
  for (int i = threadIdx.x; i < a.n; i += kThreads) a.dst[i] = a.w[i];
}
