// paged.cpp - the paged 8-bit K/V cache (llmrs_paged_*; kernels in paged.hip).
//
// The page table, each sequence's length and which pages are in use live here on
// the host, so every index a kernel reads has been checked; the device holds a
// copy of the table, which changes when pages are mapped.
#include <cmath>
#include <memory>

#include "words.h"

using namespace llmrs;

struct llmrs_paged {
  llmrs_paged_config cfg{};
  int width = 0;                 // table entries per slot
  std::vector<int> table, mapped, length;
  std::vector<char> used;        // pages
  std::vector<float> rope;       // cos, then sin; given back once on the device
  bool rotates = false;
  void *codes = nullptr, *exps = nullptr, *dtable = nullptr, *drope = nullptr;
  void* tickets = nullptr;       // of split attention tiles, zero between launches
  size_t n_tickets = 0;

  // Device memory, at the first call that needs it.
  void settle() {
    if (codes) return;
    Context& c = ctx();
    const size_t blocks = (size_t)cfg.n_pages * (cfg.page_size / kPagedBlock);
    try {
      dtable = c.alloc.alloc(4 * table.size());
      LLMRS_HIP(hipMemcpyAsync(dtable, table.data(), 4 * table.size(), hipMemcpyHostToDevice, c.stream));
      if (rotates) {
        drope = c.alloc.alloc(4 * rope.size());
        LLMRS_HIP(hipMemcpyAsync(drope, rope.data(), 4 * rope.size(), hipMemcpyHostToDevice, c.stream));
      }
      LLMRS_HIP(hipStreamSynchronize(c.stream));
      exps = c.alloc.alloc(blocks * cfg.n_kv_heads * 2);
      codes = c.alloc.alloc(blocks * paged_block_bytes(cfg.n_kv_heads, cfg.head_dim));
    } catch (...) {
      drop();
      throw;
    }
    rope.clear();
    rope.shrink_to_fit();
  }
  int* zero_tickets(size_t n) {
    if (n > n_tickets) {
      Context& c = ctx();
      if (tickets) c.alloc.release(tickets);
      tickets = nullptr;
      n_tickets = 0;
      const size_t bytes = 2 * n * kTicketStride * sizeof(int);
      tickets = c.alloc.alloc(bytes);
      LLMRS_HIP(hipMemsetAsync(tickets, 0, bytes, c.stream));
      n_tickets = 2 * n;
    }
    return (int*)tickets;
  }
  void drop() {
    for (void** p : {&codes, &exps, &dtable, &drope, &tickets}) {
      if (*p) ctx().alloc.release(*p);
      *p = nullptr;
    }
    n_tickets = 0;
  }
  int slot(int s, const char* what) const {
    LLMRS_REQUIRE(s >= 0 && s < cfg.max_seqs, LLMRS_E_RANGE,
                  std::string(what) + ": slot " + std::to_string(s) + " of " + std::to_string(cfg.max_seqs));
    return s;
  }
  PagedPool pool() const {
    return {(uint8_t*)codes, (int8_t*)exps, (const int*)dtable, width,
            __builtin_ctz((unsigned)(cfg.page_size / kPagedBlock)), cfg.n_kv_heads};
  }
  const float* cos() const { return (const float*)drope; }
  const float* sin() const { return drope ? (const float*)drope + (size_t)cfg.max_seq * (cfg.head_dim / 2) : nullptr; }
};

namespace {

std::string hd_tag(const llmrs_paged* p) { return "_hd" + std::to_string(p->cfg.head_dim); }

// One sequence of a call.
struct Part {
  int slot, row0, rows, pos;
};

// The sequences of a call: slots in range and named once, rows of a tensor of
// `rows_given` rows in the order given.  Those without rows are left out.
std::vector<Part> parts_of(const llmrs_paged* p, const int32_t* slots, const int32_t* counts, size_t n, const char* what,
                           size_t* rows) {
  LLMRS_REQUIRE((slots && counts) || !n, LLMRS_E_INVALID, std::string(what) + ": null argument");
  std::vector<char> seen((size_t)p->cfg.max_seqs);
  std::vector<Part> parts;
  size_t at = 0;
  for (size_t i = 0; i < n; ++i) {
    const int s = p->slot(slots[i], what);
    LLMRS_REQUIRE(!seen[(size_t)s], LLMRS_E_INVALID, std::string(what) + ": slot " + std::to_string(s) + " named twice");
    seen[(size_t)s] = 1;
    LLMRS_REQUIRE(counts[i] >= 0 && counts[i] <= p->cfg.max_seq, LLMRS_E_RANGE,
                  std::string(what) + ": " + std::to_string(counts[i]) + " rows in slot " + std::to_string(s));
    if (counts[i]) parts.push_back({s, (int)at, counts[i], p->length[(size_t)s]});
    at += (size_t)counts[i];
  }
  LLMRS_REQUIRE(at <= ((size_t)1 << 30), LLMRS_E_INVALID, std::string(what) + ": too many rows");
  *rows = at;
  return parts;
}

void require_rows(const llmrs_tensor* t, size_t rows, size_t width, const std::string& what) {
  LLMRS_REQUIRE(t, LLMRS_E_INVALID, what + ": null tensor");
  LLMRS_REQUIRE(t->dtype == LLMRS_F32, LLMRS_E_DTYPE, what + ": requires an f32 tensor");
  LLMRS_REQUIRE(t->dims.size() == 2 && t->dims[0] == rows && t->dims[1] == width, LLMRS_E_INVALID,
                what + ": must be [" + std::to_string(rows) + ", " + std::to_string(width) + "]");
}

// The work items of a launch, each part's; refused where `threads` of them for each item
// are more than a launch can have in one dimension (2^32 less one).
struct Items {
  std::vector<int> of;
  int total = 0;
};
template <class F>
Items count_items(const std::vector<Part>& parts, size_t threads, const char* what, F&& items) {
  Items n;
  size_t at = 0;
  for (const Part& s : parts) {
    at += items(s);
    LLMRS_REQUIRE(at * threads < ((size_t)1 << 32), LLMRS_E_INVALID, std::string(what) + ": too much work for one call");
    n.of.push_back((int)items(s));
  }
  n.total = (int)at;
  return n;
}

// What the kernels know of the parts.
std::vector<int> seq_words(const std::vector<Part>& parts, const Items& items) {
  std::vector<int> w;
  w.reserve(kPagedPerSeq * parts.size());
  int at = 0;
  for (int n : items.of) {
    w.push_back(at);
    at += n;
  }
  for (const Part& s : parts) w.insert(w.end(), {s.slot, s.row0, s.rows, s.pos});
  return w;
}

llmrs_tensor* new_rows(size_t rows, size_t width) {
  std::unique_ptr<llmrs_tensor> t(new llmrs_tensor());
  t->dims = {rows, width};
  t->bytes = rows * width * sizeof(float);
  t->data = ctx().alloc.alloc(t->bytes);
  return t.release();
}
struct TensorFree {
  void operator()(llmrs_tensor* t) const {
    ctx().alloc.release(t->data);
    delete t;
  }
};
typedef std::unique_ptr<llmrs_tensor, TensorFree> Rows;

// The blocks that the parts' rows touch.
Items row_items(const llmrs_paged* p, const std::vector<Part>& parts, const char* what) {
  return count_items(parts, 2 * (size_t)p->cfg.head_dim, what,
                     [](const Part& s) { return (size_t)(s.pos % kPagedBlock + s.rows + kPagedBlock - 1) / kPagedBlock; });
}
// One launch over them.
void launch_rows(const llmrs_paged* p, const std::string& kernel, const std::vector<Part>& parts, const Items& items,
                 float* k, float* v, bool rotate) {
  PagedRowsArgs a;
  a.pool = p->pool();
  a.rows[0] = k;
  a.rows[1] = v;
  a.rope_cos = rotate ? p->cos() : nullptr;
  a.rope_sin = rotate ? p->sin() : nullptr;
  a.seqs.n = (int)parts.size();
  a.seqs.items = items.total;
  const LaunchWords words(seq_words(parts, items), a.seqs.w);
  a.seqs.ext = words.ext();
  launch(kernel + hd_tag(p), dim3((unsigned)a.seqs.items, (unsigned)p->cfg.n_kv_heads, 2),
         dim3((unsigned)(2 * p->cfg.head_dim)), 0, ctx().stream, a);
}

// A kernel's columns per workgroup and the positions that its waves take at a time.
struct AttnKind {
  const char* name;
  int cols, unit;
};
constexpr AttnKind kFew{"few", 16, 256}, kMany{"many", 64, 64};
// Columns per CU from which the kernel of 64 is the faster: with 64 of them (512 rows
// of 32 heads behind 500 positions) 33.1 us against 28.2, with 96 (768 rows behind 1000)
// 50.1 against 51.0, with 100 (4 x 200 rows behind 1000) 43.4 against 52.7, with 256 (4 x
// 512 rows) 35.4 against 67.3 and with 256 behind 2048 positions 185 against 243.
constexpr long kManyColumns = 96;
// Positions x head_dim up to which a sequence is not split: joining takes 2.7 us, 256
// more positions in one workgroup 1.05 us with 64 dims and 2 with 128 (one row behind 512
// positions of 64 dims 7.4 us whole, 8.2 in three; behind 300 of 128 8.4 and 9.4; behind
// 1000 of 128 11.8 and 9.6).
constexpr long kWhole = 65536;

// Units of a split.  One workgroup per CU: a second one doubles what is joined for
// little (8 sequences of 4000 positions: 16.7 us with one, 16.4 with two; 64 of 1000 to
// 4000: 57 and 73).  Where that would split nothing though CUs stand half empty, two: they
// even out lengths (16 sequences of 500 to 2100 positions, two workgroups a head: 17.7 us
// against 20.1; of equal lengths 23.9 against 22.3).  A batch that fills the chip unsplit
// keeps whole sequences but for the ones that would outlast it.
int split_units(const std::vector<Part>& parts, long heads, int n_rep, int hd, const AttnKind& kind, long cus) {
  long units = 0, whole = 0;
  int longest = 0;
  auto tiles = [&](const Part& s) { return heads * ((s.rows * (long)n_rep + kind.cols - 1) / kind.cols); };
  for (const Part& s : parts) {
    units += tiles(s) * ((s.pos + kind.unit - 1) / kind.unit);
    whole += tiles(s);
    longest = std::max(longest, s.pos);
  }
  const long slots = 2 * whole > cus && whole <= cus ? 2 * cus : cus;
  const int most = (longest + kind.unit - 1) / kind.unit;
  if ((long)most * kind.unit * hd <= kWhole) return most;
  int per = (int)std::max<long>((units + slots - 1) / slots, (most + kPagedMaxSplits - 1) / kPagedMaxSplits);
  for (; whole <= slots && per < most; ++per) {
    long groups = 0;
    for (const Part& s : parts) groups += tiles(s) * ((s.pos + per * kind.unit - 1) / (per * kind.unit));
    if (groups <= slots) break;
  }
  return std::min(per, most);
}

// One launch of the attention: its sequences, kernel and splits.
struct AttnPlan {
  explicit AttnPlan(const AttnKind& k) : kind(k) {}
  AttnKind kind;
  std::vector<Part> parts;
  int chunk = 0;  // positions of a split, at most
  bool split = false;
  Items items;
  int splits(const Part& s) const { return (s.pos + chunk - 1) / chunk; }
};

// The launches of a call.  The kernel of 64 columns reads a cache a quarter as often, but
// needs columns for every CU's waves; sequences that do not fill one of its workgroups
// stay with the kernel of 16.
std::vector<AttnPlan> plan_attention(const std::vector<Part>& parts, int nkv, int n_rep, int hd, int cus) {
  AttnPlan few(kFew), many(kMany);
  long columns = 0;
  for (const Part& s : parts) {
    const bool fills = (long)s.rows * n_rep >= kMany.cols;
    (fills ? many : few).parts.push_back(s);
    if (fills) columns += (long)s.rows * n_rep * nkv;
  }
  if (columns < kManyColumns * cus) few.parts = parts, many.parts.clear();
  std::vector<AttnPlan> plans;
  for (AttnPlan* p : {&few, &many}) {
    if (p->parts.empty()) continue;
    p->chunk = split_units(p->parts, nkv, n_rep, hd, p->kind, cus) * p->kind.unit;
    p->items = count_items(p->parts, 256 * (size_t)nkv, "paged_attention", [&](const Part& s) {
      return (size_t)p->splits(s) * (((size_t)s.rows * (size_t)n_rep + (size_t)p->kind.cols - 1) / (size_t)p->kind.cols);
    });
    for (const Part& s : p->parts) p->split = p->split || p->splits(s) > 1;
    plans.push_back(std::move(*p));
  }
  return plans;
}

void launch_attention(llmrs_paged* p, const llmrs_tensor* q, llmrs_tensor* out, const AttnPlan& plan) {
  const int nkv = p->cfg.n_kv_heads, hd = p->cfg.head_dim;
  PagedAttnArgs a;
  a.pool = p->pool();
  a.q = (const float*)q->data;
  a.out = (float*)out->data;
  a.rope_cos = p->cos();
  a.rope_sin = p->sin();
  a.nq = (int)(q->dims[1] / (size_t)hd);
  a.scale = 1.0f / std::sqrt((float)hd);
  a.chunk = plan.chunk;
  a.seqs.n = (int)plan.parts.size();
  a.seqs.items = plan.items.total;
  const LaunchWords words(seq_words(plan.parts, plan.items), a.seqs.w);
  a.seqs.ext = words.ext();
  const size_t groups = (size_t)plan.items.total * (size_t)nkv;
  const size_t columns = plan.split ? groups * (size_t)plan.kind.cols : 0;
  Scratch part(columns * 4 * (size_t)(hd + 2));
  a.part_o = (float*)part.p;
  a.part_ml = a.part_o ? a.part_o + columns * (size_t)hd : nullptr;
  a.tickets = plan.split ? p->zero_tickets(groups) : nullptr;
  launch(std::string("paged_attn_") + plan.kind.name + hd_tag(p), dim3((unsigned)groups), dim3(256), 0, ctx().stream, a);
}

}  // namespace

extern "C" {

int llmrs_paged_create(const llmrs_paged_config* cfg, const float* rope_cos, const float* rope_sin, llmrs_paged** out) {
  return guard([&] {
    LLMRS_REQUIRE(cfg && out, LLMRS_E_INVALID, "paged cache: null argument");
    const llmrs_paged_config& g = *cfg;
    LLMRS_REQUIRE(g.head_dim == 64 || g.head_dim == 128, LLMRS_E_INVALID, "paged cache: head_dim must be 64 or 128");
    LLMRS_REQUIRE(g.n_kv_heads >= 1 && g.n_kv_heads <= 256, LLMRS_E_INVALID, "paged cache: n_kv_heads must be 1 to 256");
    LLMRS_REQUIRE(g.page_size >= kPagedBlock && g.page_size <= 4096 && !(g.page_size & (g.page_size - 1)), LLMRS_E_INVALID,
                  "paged cache: page_size must be a power of two from 32 to 4096");
    LLMRS_REQUIRE(g.n_pages >= 1 && (long)g.n_pages * (g.page_size / kPagedBlock) <= (1 << 30), LLMRS_E_INVALID,
                  "paged cache: n_pages out of range");
    LLMRS_REQUIRE(g.max_seqs >= 1 && g.max_seqs <= 65536, LLMRS_E_INVALID, "paged cache: max_seqs must be 1 to 65536");
    LLMRS_REQUIRE(g.max_seq >= 1 && g.max_seq <= (1 << 20), LLMRS_E_INVALID, "paged cache: max_seq must be 1 to 1048576");
    LLMRS_REQUIRE(!rope_cos == !rope_sin, LLMRS_E_INVALID, "paged cache: rope_cos and rope_sin go together");
    LLMRS_REQUIRE(g.rope_theta >= 0.0f && std::isfinite(g.rope_theta), LLMRS_E_INVALID, "paged cache: bad rope_theta");
    const int width = (g.max_seq + g.page_size - 1) / g.page_size;
    LLMRS_REQUIRE((size_t)width * (size_t)g.max_seqs <= ((size_t)1 << 28), LLMRS_E_INVALID,
                  "paged cache: max_seqs * max_seq / page_size exceeds 2^28 table entries");
    std::unique_ptr<llmrs_paged> p(new llmrs_paged());
    p->cfg = g;
    p->width = width;
    p->table.assign((size_t)width * (size_t)g.max_seqs, -1);
    p->mapped.assign((size_t)g.max_seqs, 0);
    p->length.assign((size_t)g.max_seqs, 0);
    p->used.assign((size_t)g.n_pages, 0);
    const size_t half = (size_t)g.max_seq * (size_t)(g.head_dim / 2);
    p->rotates = rope_cos || g.rope_theta > 0.0f;
    if (p->rotates) {
      p->rope.resize(2 * half);
      if (rope_cos) {
        std::copy(rope_cos, rope_cos + half, p->rope.begin());
        std::copy(rope_sin, rope_sin + half, p->rope.begin() + (long)half);
      } else {
        rope_table(0, (size_t)g.max_seq, g.head_dim, g.rope_theta, p->rope.data(), p->rope.data() + half);
      }
    }
    *out = p.release();
  });
}

int llmrs_paged_free(llmrs_paged* p) {
  return guard([&] {
    if (!p) return;
    if (p->codes) p->drop();
    delete p;
  });
}

int llmrs_paged_map(llmrs_paged* p, int32_t slot, const int32_t* pages, size_t n) {
  return guard([&] {
    LLMRS_REQUIRE(p && (pages || !n), LLMRS_E_INVALID, "paged_map: null argument");
    const size_t s = (size_t)p->slot(slot, "paged_map"), at = (size_t)p->mapped[s];
    LLMRS_REQUIRE(n <= (size_t)p->width - at, LLMRS_E_RANGE,
                  "paged_map: slot " + std::to_string(slot) + " holds at most " + std::to_string(p->width) + " pages");
    size_t taken = 0;  // pages marked so far, given back if one cannot be had
    try {
      for (; taken < n; ++taken) {
        const int page = pages[taken];
        LLMRS_REQUIRE(page >= 0 && page < p->cfg.n_pages, LLMRS_E_RANGE,
                      "paged_map: page " + std::to_string(page) + " of " + std::to_string(p->cfg.n_pages));
        LLMRS_REQUIRE(!p->used[(size_t)page], LLMRS_E_INVALID, "paged_map: page " + std::to_string(page) + " is in use");
        p->used[(size_t)page] = 1;
      }
      if (p->codes && n) {
        OnDevice here;
        set_words((int*)p->dtable + s * (size_t)p->width + at, pages, n);
      }
    } catch (...) {
      while (taken) p->used[(size_t)pages[--taken]] = 0;
      throw;
    }
    std::copy(pages, pages + n, &p->table[s * (size_t)p->width + at]);
    p->mapped[s] += (int)n;
  });
}

int llmrs_paged_release(llmrs_paged* p, int32_t slot) {
  return guard([&] {
    LLMRS_REQUIRE(p, LLMRS_E_INVALID, "paged_release: null argument");
    const size_t s = (size_t)p->slot(slot, "paged_release");
    for (int i = 0; i < p->mapped[s]; ++i) {
      int& page = p->table[s * (size_t)p->width + (size_t)i];
      p->used[(size_t)page] = 0;
      page = -1;
    }
    p->mapped[s] = p->length[s] = 0;
  });
}

int llmrs_paged_length(const llmrs_paged* p, int32_t slot, int32_t* length) {
  return guard([&] {
    LLMRS_REQUIRE(p && length, LLMRS_E_INVALID, "paged_length: null argument");
    *length = p->length[(size_t)p->slot(slot, "paged_length")];
  });
}

int llmrs_paged_truncate(llmrs_paged* p, const int32_t* slots, const int32_t* lengths, size_t n) {
  return guard([&] {
    LLMRS_REQUIRE(p && ((slots && lengths) || !n), LLMRS_E_INVALID, "paged_truncate: null argument");
    std::vector<char> seen((size_t)p->cfg.max_seqs);
    for (size_t i = 0; i < n; ++i) {
      const size_t s = (size_t)p->slot(slots[i], "paged_truncate");
      LLMRS_REQUIRE(!seen[s], LLMRS_E_INVALID, "paged_truncate: slot " + std::to_string(s) + " named twice");
      seen[s] = 1;
      const int have = p->length[s];
      LLMRS_REQUIRE(lengths[i] >= 0 && lengths[i] <= have, LLMRS_E_RANGE,
                    "paged_truncate: " + std::to_string(lengths[i]) + " positions of " + std::to_string(have) + " in slot " +
                        std::to_string(slots[i]));
    }
    for (size_t i = 0; i < n; ++i) p->length[(size_t)slots[i]] = lengths[i];
  });
}

int llmrs_paged_append(llmrs_paged* p, const llmrs_tensor* k, const llmrs_tensor* v, const int32_t* slots,
                       const int32_t* counts, size_t n, int rotate) {
  return guard([&] {
    LLMRS_REQUIRE(p, LLMRS_E_INVALID, "paged_append: null argument");
    size_t rows = 0;
    const std::vector<Part> parts = parts_of(p, slots, counts, n, "paged_append", &rows);
    const size_t width = (size_t)p->cfg.n_kv_heads * (size_t)p->cfg.head_dim;
    for (const Part& s : parts) {
      const long end = (long)s.pos + s.rows;
      LLMRS_REQUIRE(end <= p->cfg.max_seq && end <= (long)p->mapped[(size_t)s.slot] * p->cfg.page_size, LLMRS_E_RANGE,
                    "paged_append: slot " + std::to_string(s.slot) + " has no page for position " + std::to_string(end - 1));
    }
    const Items items = row_items(p, parts, "paged_append");
    require_rows(k, rows, width, "paged_append k");
    require_rows(v, rows, width, "paged_append v");
    if (parts.empty()) return;
    (void)ctx();
    OnDevice here;
    p->settle();
    launch_rows(p, "paged_append", parts, items, (float*)k->data, (float*)v->data, rotate != 0);
    for (const Part& s : parts) p->length[(size_t)s.slot] += s.rows;
  });
}

int llmrs_paged_read(llmrs_paged* p, const int32_t* slots, const int32_t* starts, const int32_t* counts, size_t n,
                     llmrs_tensor** k, llmrs_tensor** v) {
  return guard([&] {
    LLMRS_REQUIRE(p && k && v && (starts || !n), LLMRS_E_INVALID, "paged_read: null argument");
    size_t rows = 0, i = 0;
    std::vector<Part> parts = parts_of(p, slots, counts, n, "paged_read", &rows);
    for (size_t s = 0; s < n; ++s) {
      LLMRS_REQUIRE(starts[s] >= 0 && (long)starts[s] + counts[s] <= p->length[(size_t)slots[s]], LLMRS_E_RANGE,
                    "paged_read: positions " + std::to_string(starts[s]) + " to " + std::to_string((long)starts[s] + counts[s]) +
                        " of " + std::to_string(p->length[(size_t)slots[s]]) + " in slot " + std::to_string(slots[s]));
      if (counts[s]) parts[i++].pos = starts[s];
    }
    const Items items = row_items(p, parts, "paged_read");
    (void)ctx();
    OnDevice here;
    const size_t width = (size_t)p->cfg.n_kv_heads * (size_t)p->cfg.head_dim;
    Rows kr(new_rows(rows, width)), vr(new_rows(rows, width));
    if (!parts.empty()) launch_rows(p, "paged_read", parts, items, (float*)kr->data, (float*)vr->data, false);
    *k = kr.release();
    *v = vr.release();
  });
}

int llmrs_paged_attention(llmrs_paged* p, const llmrs_tensor* q, const int32_t* slots, const int32_t* counts, size_t n,
                          llmrs_tensor** out) {
  return guard([&] {
    LLMRS_REQUIRE(p && out, LLMRS_E_INVALID, "paged_attention: null argument");
    size_t rows = 0;
    const std::vector<Part> parts = parts_of(p, slots, counts, n, "paged_attention", &rows);
    for (const Part& s : parts)
      LLMRS_REQUIRE(s.rows <= s.pos, LLMRS_E_RANGE,
                    "paged_attention: " + std::to_string(s.rows) + " rows of " + std::to_string(s.pos) + " positions in slot " +
                        std::to_string(s.slot));
    LLMRS_REQUIRE(q, LLMRS_E_INVALID, "paged_attention q: null tensor");
    const size_t group = (size_t)p->cfg.n_kv_heads * (size_t)p->cfg.head_dim;
    LLMRS_REQUIRE(q->dims.size() == 2 && q->dims[1] > 0 && q->dims[1] % group == 0 && q->dims[1] <= 65536, LLMRS_E_INVALID,
                  "paged_attention: q must be [rows, query heads * head_dim] with whole groups of query heads");
    require_rows(q, rows, q->dims[1], "paged_attention q");
    OnDevice here;
    const std::vector<AttnPlan> plans =
        plan_attention(parts, p->cfg.n_kv_heads, (int)(q->dims[1] / group), p->cfg.head_dim, ctx().num_cus);
    Rows o(new_rows(rows, q->dims[1]));
    for (const AttnPlan& plan : plans) launch_attention(p, q, o.get(), plan);
    *out = o.release();
  });
}

int llmrs_probe_paged_plan(int n_kv_heads, int head_dim, int group, const int32_t* lengths, const int32_t* counts, size_t n,
                           int num_cus, int32_t* columns, int32_t* splits) {
  return guard([&] {
    LLMRS_REQUIRE(lengths && counts && columns && splits, LLMRS_E_INVALID, "probe_paged_plan: null argument");
    LLMRS_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 256 && (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 1024 &&
                      num_cus > 0 && n <= 65536, LLMRS_E_INVALID, "probe_paged_plan: bad argument");
    std::vector<Part> parts;
    for (size_t i = 0; i < n; ++i) {
      LLMRS_REQUIRE(counts[i] >= 0 && counts[i] <= lengths[i] && lengths[i] <= (1 << 20), LLMRS_E_RANGE,
                    "probe_paged_plan: bad length");
      columns[i] = splits[i] = 0;
      if (counts[i]) parts.push_back({(int)i, 0, counts[i], lengths[i]});
    }
    for (const AttnPlan& plan : plan_attention(parts, n_kv_heads, group, head_dim, num_cus))
      for (const Part& s : plan.parts) {
        columns[s.slot] = plan.kind.cols;
        splits[s.slot] = plan.splits(s);
      }
  });
}

}  // extern "C"
