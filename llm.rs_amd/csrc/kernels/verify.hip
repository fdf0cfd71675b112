// verify.hip - drafted tokens against the target's probabilities, from given
// random numbers, for gfx950.
//
// No counterpart in the reference, which draws one token per forward
// (src/main.rs:192-305).  Draft j of a sequence, id x with target probability
// p(x) and draft probability q(x), is accepted while u_j q(x) < p(x): the product
// of two f32 values is exact in 64 bits, so no rounding decides.  The first
// refusal draws from max(p - q, 0), a sequence without one from the target row
// after its last draft: the smallest id whose running sum exceeds draw * total.
// The sums are 64 bits and of one order (eight ids of a lane in turn, the lanes and
// then the slices as trees), so the id is that of the formula where the draw does not
// meet a running sum to within their roundings, and always one that has something.
// Where nothing is left of the target, it is drawn from as it is.
#include "common.h"
#include "../kernel_args.h"

using namespace llmrs;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / LLMRS_WAVE;
constexpr int kPer = kVerifySlice / LLMRS_WAVE;  // ids per lane of a slice, consecutive
constexpr int kHeld = 8;                         // sums of the slices, 64 at a time, that a wave holds

__device__ __forceinline__ int word(const VerifyArgs& a, int i) { return a.ext ? a.ext[i] : a.w[i]; }

struct Row {
  int accepted, drafts, first, drafted;  // first: its drafts in the list; drafted: the refused id (-1: none)
  const float* p;
  const float* q;  // null: none, or one id only
};
// How many drafts of sequence i are accepted, and the rows its next token is
// drawn from.  One draft per lane.
__device__ __forceinline__ Row examine(const VerifyArgs& a, int i) {
  Row r;
  // (one value per wave: the compiler takes what is loaded from either of two places
  // to differ from lane to lane)
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int row = uni(word(a, 3 * i));
  r.first = uni(word(a, 3 * i + 1));
  r.drafts = uni(word(a, 3 * i + 2));
  const int lane = lane_id(), base = 3 * a.n + r.first;
  bool refused = false;
  if (lane < r.drafts) {
    const int id = word(a, base + lane);
    const double u = __int_as_float(word(a, base + a.drafts + lane));
    const double p = a.target[(size_t)(row + lane) * a.vocab + id];
    const double q = a.draft ? a.draft[(size_t)(r.first + lane) * a.vocab + id] : 1.0f;
    refused = !(u * q < p);
  }
  const unsigned long long mask = __ballot(refused);
  r.accepted = mask ? __builtin_ctzll(mask) : r.drafts;
  r.p = a.target + (size_t)(row + r.accepted) * a.vocab;
  const bool rest = r.accepted < r.drafts;
  r.q = rest && a.draft ? a.draft + (size_t)(r.first + r.accepted) * a.vocab : nullptr;
  r.drafted = rest && !a.draft ? uni(word(a, base + r.accepted)) : -1;
  return r;
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any id

// The weights of this thread's ids v0 .. v0 + 7: what is left of the target, or the
// target itself; NaN counts as zero, ids past the vocabulary too.
template <bool LEFT>
__device__ __forceinline__ void weights(const VerifyArgs& a, const Row& r, int v0, double (&w)[kPer]) {
  float p[kPer], q[kPer];
  if (v0 + kPer <= a.vocab) {
#pragma unroll
    for (int k = 0; k < kPer; k += 4) {
      const f32x4u x = *(const f32x4u*)(r.p + v0 + k);
      f32x4u y = {0.0f, 0.0f, 0.0f, 0.0f};
      if (LEFT && r.q) y = *(const f32x4u*)(r.q + v0 + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[k + i] = x[i];
        q[k + i] = y[i];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      p[k] = v0 + k < a.vocab ? r.p[v0 + k] : 0.0f;
      q[k] = LEFT && r.q && v0 + k < a.vocab ? r.q[v0 + k] : 0.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (LEFT && v0 + k == r.drafted) q[k] = 1.0f;
    const double x = (double)p[k] - (LEFT ? (double)q[k] : 0.0);
    w[k] = x > 0.0 ? x : 0.0;
  }
}

// Inclusive running sum over the lanes (row shifts, then the rows' last lanes
// broadcast); lane 63 holds the total.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double v) {
  const dev_u32x2 u = __builtin_bit_cast(dev_u32x2, v);
  const dev_u32x2 r = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)u.x, CTRL, ROWS, 0xF, false),
                       (unsigned)__builtin_amdgcn_update_dpp(0, (int)u.y, CTRL, ROWS, 0xF, false)};
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double scan(double v) {
  v += dpp64<0x111, 0xF>(v);  // row_shr:1, zero where the row begins
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp64<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const dev_u32x2 u = __builtin_bit_cast(dev_u32x2, v);
  const dev_u32x2 r = {(unsigned)__builtin_amdgcn_readlane((int)u.x, lane), (unsigned)__builtin_amdgcn_readlane((int)u.y, lane)};
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ int last_of(unsigned long long mask) { return 63 - __builtin_clzll(mask); }

// A slice's ids by one wave: the sum, and where the running sum from `base` exceeds
// tau (-1: nowhere) and the last id that holds anything (-1: none).
template <bool LEFT>
__device__ __forceinline__ double slice_sum(const VerifyArgs& a, const Row& r, int slice, double (&w)[kPer]) {
  weights<LEFT>(a, r, slice * kVerifySlice + lane_id() * kPer, w);
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) sum += w[k];
  return scan(sum);
}
template <bool LEFT>
__device__ __forceinline__ void slice_draw(const VerifyArgs& a, const Row& r, int slice, double base, double tau, int* id,
                                           int* last) {
  double w[kPer];
  const double incl = slice_sum<LEFT>(a, r, slice, w);
  double c = base + dpp64<0x138, 0xF>(incl);  // wave_shr:1: the lanes before
  int hit = -1, top = -1;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    c += w[k];
    if (w[k] > 0.0) {
      top = k;
      if (hit < 0 && c > tau) hit = k;
    }
  }
  const int v0 = slice * kVerifySlice;
  const unsigned long long hits = __ballot(hit >= 0), tops = __ballot(top >= 0);
  const int hl = hits ? __builtin_ctzll(hits) : 0, tl = tops ? last_of(tops) : 0;
  *id = hits ? v0 + hl * kPer + __builtin_amdgcn_readlane(hit, hl) : -1;
  *last = tops ? v0 + tl * kPer + __builtin_amdgcn_readlane(top, tl) : -1;
}

// The draw of a sequence, by one wave: `part` holds the slices' sums of what is
// left of the target.
__device__ __forceinline__ int draw(const VerifyArgs& a, const Row& r, const unsigned* part, double u) {
  const int lane = lane_id(), groups = a.groups;
  double x[kHeld];  // running sums of 64 slices each
  // the slices that hold anything: the running sums are formed as trees, so one may
  // rise by a last place past a slice that does not
  unsigned long long some[kHeld];
  auto hold = [&](int g0) {
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      const int g = g0 + LLMRS_WAVE * c + lane;
      x[c] = g < groups ? __builtin_bit_cast(double, dev_ld8(part, 8 * g)) : 0.0;
    }
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      some[c] = __ballot(x[c] > 0.0);
      if (g0 + LLMRS_WAVE * c < groups) x[c] = scan(x[c]);
    }
  };
  constexpr int HELD = LLMRS_WAVE * kHeld;
  double total = 0.0;
  for (int g0 = 0; g0 < groups; g0 += HELD) {
    hold(g0);
#pragma unroll
    for (int c = 0; c < kHeld; ++c) total += lane64(x[c], 63);
  }
  int id = -1, last = -1;
  if (!(total > 0.0)) {
    // nothing is left of the target (rare): the target itself, slice by slice
    double w[kPer];
    for (int g = 0; g < groups; ++g) total += lane64(slice_sum<false>(a, r, g, w), 63);
    const double tau = u * total;
    double base = 0.0;
    for (int g = 0; g < groups && id < 0; ++g) {
      const double sum = lane64(slice_sum<false>(a, r, g, w), 63);
      if (sum > 0.0) {
        int top;
        slice_draw<false>(a, r, g, base, tau, &id, &top);
        last = top;
      }
      base += sum;
    }
    return id >= 0 ? id : last >= 0 ? last : a.vocab - 1;
  }
  // the first slice whose running sum exceeds tau, or the last that holds anything
  const double tau = u * total;
  double base = 0.0, from = 0.0;
  int slice = -1, top = 0;
  for (int g0 = 0; g0 < groups && slice < 0; g0 += HELD) {
    if (groups > HELD) hold(g0);
#pragma unroll
    for (int c = 0; c < kHeld; ++c) {
      if (g0 + LLMRS_WAVE * c >= groups) break;
      const unsigned long long over = __ballot(base + x[c] > tau) & some[c];
      const double before = dpp64<0x138, 0xF>(x[c]);
      if (slice < 0 && over) {
        const int l = __builtin_ctzll(over);
        slice = g0 + LLMRS_WAVE * c + l;
        from = base + lane64(before, l);
      }
      if (slice < 0 && some[c]) top = g0 + LLMRS_WAVE * c + last_of(some[c]);
      base += lane64(x[c], 63);
    }
  }
  // sums in another order may end just below what crossed: the slice's last id
  if (slice >= 0) slice_draw<true>(a, r, slice, from, tau, &id, &last);
  else slice_draw<true>(a, r, top, 0.0, INFINITY, &id, &last);
  return id >= 0 ? id : last >= 0 ? last : a.vocab - 1;
}

}  // namespace

// A wave sums slices of a sequence's row.  The sequence's last workgroup (a ticket, no
// waiting; the sums move with device-scope stores and loads) draws, one wave of it
// alone: the slice in which the running sum crosses, and the id in that slice.  Its
// answer goes straight to the host's memory, where the caller waits for the stamps.
// Bound by latency (words, drafted ids, row, sums, ticket, sums, slice): 5.9 us (median
// of 125 launches; the fastest 5.5) for one sequence of 32000 ids, 8.3 us (7.7) for 32 of
// 128256 with drafts' probabilities (33 MB); tickets next to each other in memory made
// that 34.
extern "C" __global__ __launch_bounds__(kThreads) void verify_rows(VerifyArgs a) {
  const int i = blockIdx.y, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(wave_id());
  const Row r = examine(a, i);
  unsigned* part = (unsigned*)(a.part + (size_t)i * a.groups);
  const int first = blockIdx.x * kWaves * a.per_wave + wave, end = min(first + kWaves * a.per_wave, a.groups);
  for (int g = first; g < end; g += kWaves) {
    double w[kPer];
    const double sum = slice_sum<true>(a, r, g, w);
    if (lane_id() == 63) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(dev_u32x2, sum), dev_rsrc(part), 8 * g, 0, kSc1);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (wave) return;
  int ticket = 0;
  if (tid == 0) ticket = atomicAdd(a.tickets + (size_t)i * kTicketStride, 1);
  if (__builtin_amdgcn_readfirstlane(ticket) != (int)gridDim.x - 1) return;
  if (tid == 0) dev_stu(a.tickets + (size_t)i * kTicketStride, 0, 0u);  // as it was found, for the next launch
  const int drawn = draw(a, r, part, __int_as_float(word(a, 3 * a.n + 2 * a.drafts + i)));
  // to the host's memory, each word with its stamp, so nothing waits for another
  unsigned long long* out = a.out + (size_t)i * (a.most + 2);
  for (int j = tid; j < a.most + 2; j += LLMRS_WAVE) {
    const int at = j - 1;  // accepted drafts, tokens
    const int v = j == 0 ? r.accepted : at < r.accepted ? word(a, 3 * a.n + r.first + at) : at == r.accepted ? drawn : -1;
    __hip_atomic_store(out + j, (unsigned long long)kVerifyStamp << 32 | (unsigned)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}
