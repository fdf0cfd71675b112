// verify.hip - drafted tokens against the target's probabilities, from given
// random numbers, for gfx950.
//
// No counterpart in the reference, which draws one token per forward
// (src/main.rs:192-305).  Draft j of a sequence, id x with target probability
// p(x) and draft probability q(x), is accepted while u_j q(x) < p(x): the product
// of two f32 values is exact in 64 bits, so no rounding decides.  The first
// refusal draws from max(p - q, 0), a sequence without one from the target row
// after its last draft: the smallest id whose running sum (64 bits, index order)
// exceeds draw * total.  Where nothing is left of the target, it is drawn from as
// it is.
#include "common.h"
#include "../kernel_args.h"

using namespace llmrs;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / LLMRS_WAVE;
constexpr int kPer = kVerifySlice / kThreads;  // ids per thread, consecutive

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
  const int row = word(a, 3 * i);
  r.first = word(a, 3 * i + 1);
  r.drafts = word(a, 3 * i + 2);
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
  r.drafted = rest && !a.draft ? word(a, base + r.accepted) : -1;
  return r;
}

// What is left of the target at id v, and the target (NaN counts as zero).
__device__ __forceinline__ double weight(const Row& r, int v, double* target) {
  const double p = r.p[v], q = r.q ? r.q[v] : v == r.drafted ? 1.0f : 0.0f;
  *target = p > 0.0 ? p : 0.0;
  const double w = p - q;
  return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Exclusive prefix over the workgroup's threads, and the total.
__device__ double prefix(double v, double* red, double* total) {
  double incl = v;
#pragma unroll
  for (int o = 1; o < LLMRS_WAVE; o <<= 1) {
    const double t = __shfl_up(incl, o);
    if (lane_id() >= o) incl += t;
  }
  if (lane_id() == LLMRS_WAVE - 1) red[wave_id()] = incl;
  __syncthreads();
  double base = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave_id()) base += red[w];
    all += red[w];
  }
  __syncthreads();
  *total = all;
  return base + (incl - v);
}

}  // namespace

// The sums of one slice of a sequence's row.
extern "C" __global__ __launch_bounds__(kThreads) void verify_sums(VerifyArgs a) {
  __shared__ double red[2][kWaves];
  const int i = blockIdx.y, g = blockIdx.x;
  const Row r = examine(a, i);
  double left = 0.0, all = 0.0;
  for (int v = g * kVerifySlice + threadIdx.x, n = 0; n < kPer; v += kThreads, ++n)
    if (v < a.vocab) {
      double t;
      left += weight(r, v, &t);
      all += t;
    }
  left = wave_sum64(left);
  all = wave_sum64(all);
  if (lane_id() == 0) {
    red[0][wave_id()] = left;
    red[1][wave_id()] = all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double* dst = a.part + 2 * ((size_t)i * a.groups + g);
    dst[0] = ((red[0][0] + red[0][1]) + red[0][2]) + red[0][3];
    dst[1] = ((red[1][0] + red[1][1]) + red[1][2]) + red[1][3];
  }
}

// The draw of one sequence: the slice that the running sum crosses in, then the id.
extern "C" __global__ __launch_bounds__(kThreads) void verify_pick(VerifyArgs a) {
  __shared__ double red[kWaves];
  __shared__ int found, last;
  __shared__ double before;
  const int i = blockIdx.x, tid = threadIdx.x;
  const Row r = examine(a, i);
  const double* part = a.part + 2 * (size_t)i * a.groups;
  const double u = __int_as_float(word(a, 3 * a.n + 2 * a.drafts + i));
  // groups in index order, consecutive ones per thread
  const int per = (a.groups + kThreads - 1) / kThreads;
  const int g0 = min(a.groups, tid * per), g1 = min(a.groups, g0 + per);
  double mine = 0.0, total;
  for (int g = g0; g < g1; ++g) mine += part[2 * g];
  double base = prefix(mine, red, &total);
  const int which = total > 0.0 ? 0 : 1;
  if (which) {
    mine = 0.0;
    for (int g = g0; g < g1; ++g) mine += part[2 * g + 1];
    base = prefix(mine, red, &total);
  }
  const double tau = u * total;
  if (tid == 0) {
    found = 0x7FFFFFFF;
    last = -1;
  }
  __syncthreads();
  int hit = -1;
  double hit_base = 0.0;
  for (int g = g0; g < g1; ++g) {
    const double w = part[2 * g + which];
    if (hit < 0 && base + w > tau) {
      hit = g;
      hit_base = base;
    }
    if (w > 0.0) atomicMax(&last, g);
    base += w;
  }
  if (hit >= 0) atomicMin(&found, hit);
  __syncthreads();
  // no slice crosses (rounding): the last one that holds anything
  const int group = found != 0x7FFFFFFF ? found : last;
  if (hit == group && hit >= 0) before = hit_base;
  __syncthreads();
  const bool end = found == 0x7FFFFFFF;
  const double from = end ? 0.0 : before;
  __syncthreads();
  if (tid == 0) {
    found = 0x7FFFFFFF;
    last = -1;
  }
  __syncthreads();
  if (group >= 0) {
    const int v0 = group * kVerifySlice + tid * kPer;
    double w[kPer], sum = 0.0, all;
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      double t = 0.0, l = 0.0;
      if (v0 + n < a.vocab) l = weight(r, v0 + n, &t);
      w[n] = which ? t : l;
      sum += w[n];
    }
    double c = from + prefix(sum, red, &all);
    int id = -1, top = -1;
#pragma unroll
    for (int n = 0; n < kPer; ++n) {
      c += w[n];
      if (w[n] > 0.0) {
        top = v0 + n;
        if (id < 0 && !end && c > tau) id = v0 + n;
      }
    }
    if (id >= 0) atomicMin(&found, id);
    if (top >= 0) atomicMax(&last, top);
  }
  __syncthreads();
  // the running sum of one order may end just below what another crossed: the last id
  const int drawn = found != 0x7FFFFFFF ? found : last >= 0 ? last : a.vocab - 1;
  int* out = a.out + (size_t)i * (a.most + 2);
  if (tid == 0) out[0] = r.accepted;
  for (int j = tid; j <= a.most; j += kThreads)
    out[1 + j] = j < r.accepted ? word(a, 3 * a.n + r.first + j) : j == r.accepted ? drawn : -1;
}
