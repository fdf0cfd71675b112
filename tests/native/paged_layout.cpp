// paged_layout.cpp - test helper: every code of a block of the paged cache has a
// place of its own, and the matrix-core operands find them where they are.
#include <cstdio>
#include <vector>

#include "kernel_args.h"

using namespace llmrs;

int main() {
  int bad = 0;
  for (int hd : {64, 128}) {
    std::vector<int> k(kPagedBlock * hd), v(kPagedBlock * hd);
    for (int p = 0; p < kPagedBlock; ++p)
      for (int d = 0; d < hd; ++d) {
        const int ko = paged_k_offset(p, d, hd), vo = paged_v_offset(p, d);
        if (ko < 0 || ko >= kPagedBlock * hd || vo < 0 || vo >= kPagedBlock * hd) return std::printf("out of the block\n"), 1;
        ++k[ko];
        ++v[vo];
      }
    for (int n : k) bad += n != 1;
    for (int n : v) bad += n != 1;
    // lane (c, r) of K operand rows b, step s: 16 bytes at b, s, r and c % 8 of the
    // block c / 8 of a 64-position tile; its row is position 16 (c / 4) + 4 b + c % 4
    for (int b = 0; b < 4; ++b)
      for (int s = 0; s < hd / 64; ++s)
        for (int c = 0; c < 16; ++c)
          for (int r = 0; r < 4; ++r)
            for (int e = 0; e < 16; ++e) {
              const int pos = 16 * (c / 4) + 4 * b + c % 4;
              const int d = hd == 128 ? 64 * s + 16 * r + e : (e & 7) + 8 * r + (e >> 3) * 32;
              bad += pos / kPagedBlock != c / 8;
              bad += paged_k_offset(pos % kPagedBlock, d, hd) != (b * (hd / 64) + s) * 512 + r * 128 + (c & 7) * 16 + e;
            }
    // lane (c, r) of V dims 16 d .. 16 d + 15: 16 positions from 16 r on
    for (int d = 0; d < hd / 16; ++d)
      for (int c = 0; c < 16; ++c)
        for (int r = 0; r < 4; ++r)
          for (int e = 0; e < 16; ++e)
            bad += paged_v_offset((16 * r + e) % kPagedBlock, 16 * d + c) != d * 512 + (r & 1) * 256 + c * 16 + e;
  }
  std::printf("mismatches %d\n", bad);
  return bad != 0;
}
