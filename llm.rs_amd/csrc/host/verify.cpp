// verify.cpp - llmrs_verify_drafts: drafted tokens against the target's
// probabilities (verify.hip).
#include <chrono>
#include <cstring>

#include "words.h"

using namespace llmrs;

namespace {

void require_rows(const llmrs_tensor* t, size_t rows, size_t vocab, const char* what) {
  LLMRS_REQUIRE(t->dtype == LLMRS_F32, LLMRS_E_DTYPE, std::string("verify_drafts: ") + what + " must be an f32 tensor");
  LLMRS_REQUIRE(t->dims.size() == 2 && t->dims[0] == rows && t->dims[1] == vocab, LLMRS_E_INVALID,
                std::string("verify_drafts: ") + what + " must be [" + std::to_string(rows) + ", " + std::to_string(vocab) + "]");
}

// Waits until every word bears the stamp.  The host sees them about 5 us before
// hipStreamSynchronize returns (an empty kernel, launch to return: 6.6 against 11.5
// us); work that is not done within a millisecond is waited for there.
void wait_for_stamps(const uint64_t* words, size_t n) {
  const auto until = std::chrono::steady_clock::now() + std::chrono::milliseconds(1);
  auto there = [&](size_t i) { return __atomic_load_n(words + i, __ATOMIC_ACQUIRE) >> 32 == kVerifyStamp; };
  for (size_t i = 0; i < n;) {
    if (there(i)) ++i;
    else if (std::chrono::steady_clock::now() > until) break;
  }
  for (size_t i = 0; i < n; ++i)
    if (!there(i)) {
      LLMRS_HIP(hipStreamSynchronize(ctx().stream));
      LLMRS_REQUIRE(there(i), LLMRS_E_HIP, "verify_drafts: no answer");
    }
}

}  // namespace

extern "C" int llmrs_verify_drafts(const llmrs_tensor* target, const llmrs_tensor* draft, const int32_t* ids,
                                   const int32_t* counts, const float* accept, const float* draw, size_t n,
                                   int32_t* accepted, int32_t* tokens, size_t width) {
  return guard([&] {
    if (!n) return;
    LLMRS_REQUIRE(target && counts && draw && accepted && tokens, LLMRS_E_INVALID, "verify_drafts: null argument");
    LLMRS_REQUIRE(n <= 65535, LLMRS_E_INVALID, "verify_drafts: at most 65535 sequences");
    LLMRS_REQUIRE(target->dims.size() == 2 && target->dims[1] > 0 && target->dims[1] <= ((size_t)1 << 30), LLMRS_E_INVALID,
                  "verify_drafts: target must be [rows, vocabulary]");
    const size_t vocab = target->dims[1];
    size_t total = 0, most = 0;
    std::vector<int> w(3 * n);
    for (size_t i = 0; i < n; ++i) {
      LLMRS_REQUIRE(counts[i] >= 0 && counts[i] <= kVerifyMaxDrafts, LLMRS_E_RANGE,
                    "verify_drafts: sequence " + std::to_string(i) + " has " + std::to_string(counts[i]) + " drafts (0 to " +
                        std::to_string(kVerifyMaxDrafts) + ")");
      w[3 * i] = (int)(total + i);
      w[3 * i + 1] = (int)total;
      w[3 * i + 2] = counts[i];
      total += (size_t)counts[i];
      most = std::max(most, (size_t)counts[i]);
    }
    require_rows(target, total + n, vocab, "target");
    if (draft) require_rows(draft, total, vocab, "draft");
    LLMRS_REQUIRE(!total || (ids && accept), LLMRS_E_INVALID, "verify_drafts: null argument");
    LLMRS_REQUIRE(width > most, LLMRS_E_INVALID,
                  "verify_drafts: rows of " + std::to_string(width) + " tokens cannot hold " + std::to_string(most) +
                      " drafts and the next token");
    for (size_t j = 0; j < total; ++j) {
      LLMRS_REQUIRE(ids[j] >= 0 && (size_t)ids[j] < vocab, LLMRS_E_RANGE,
                    "verify_drafts: drafted id " + std::to_string(ids[j]) + " outside the vocabulary");
      LLMRS_REQUIRE(accept[j] >= 0.0f && accept[j] <= 1.0f, LLMRS_E_INVALID, "verify_drafts: accept outside [0, 1]");
    }
    for (size_t i = 0; i < n; ++i)
      LLMRS_REQUIRE(draw[i] >= 0.0f && draw[i] < 1.0f, LLMRS_E_INVALID, "verify_drafts: draw outside [0, 1)");
    Context& c = ctx();
    OnDevice here;
    w.insert(w.end(), ids, ids + total);
    const size_t at = w.size();
    w.resize(at + total + n);
    if (total) std::memcpy(&w[at], accept, 4 * total);
    std::memcpy(&w[at + total], draw, 4 * n);

    VerifyArgs a;
    a.target = (const float*)target->data;
    a.draft = draft ? (const float*)draft->data : nullptr;
    a.vocab = (int)vocab;
    a.n = (int)n;
    a.groups = verify_groups((int)vocab);
    a.most = (int)most;
    a.drafts = (int)total;
    const size_t row = 2 + most, bytes = 8 * n * row;
    // tickets: zeroed here, and by each sequence's last workgroup
    if (c.n_verify_tickets < n) {
      if (c.verify_tickets) c.alloc.release(c.verify_tickets);
      c.verify_tickets = nullptr;
      c.n_verify_tickets = 0;
      const size_t size = 2 * n * kTicketStride * sizeof(int);
      c.verify_tickets = c.alloc.alloc(size);
      LLMRS_HIP(hipMemsetAsync(c.verify_tickets, 0, size, c.stream));
      c.n_verify_tickets = 2 * n;
    }
    const bool direct = bytes <= kFetchBytes;  // else through device memory
    Scratch part(8 * n * (size_t)a.groups), out(direct ? 0 : bytes);
    a.part = (double*)part.p;
    a.tickets = (int*)c.verify_tickets;
    a.out = direct ? (unsigned long long*)c.host_out : (unsigned long long*)out.p;
    // slices per wave: as many as leave four workgroups per CU; each looks at all
    // of its sequence's drafts first
    const size_t groups4 = ((size_t)a.groups + 3) / 4;
    a.per_wave = (int)std::max<size_t>(1, n * groups4 / (4 * (size_t)c.num_cus));
    const unsigned grid = (unsigned)((groups4 + a.per_wave - 1) / a.per_wave);
    if (direct)
      for (size_t i = 0; i < n * row; ++i) __atomic_store_n((uint64_t*)c.host_out + i, 0, __ATOMIC_RELAXED);
    LaunchWords words(w, a.w);
    a.ext = words.ext();
    launch("verify_rows", dim3(grid, (unsigned)n), dim3(256), 0, c.stream, a);
    std::vector<uint64_t> big;
    const uint64_t* got = (const uint64_t*)c.host_out;
    if (direct) {
      wait_for_stamps(got, n * row);
    } else {
      big.resize(n * row);
      fetch(big.data(), out.p, bytes);
      got = big.data();
    }
    for (size_t i = 0; i < n; ++i) {
      accepted[i] = (int32_t)got[i * row];
      for (size_t j = 0; j < width; ++j) tokens[i * width + j] = j <= most ? (int32_t)got[i * row + 1 + j] : -1;
    }
  });
}
