// The split of tree attention's batches over workers, as tree_split walks it: the checks
// of share_check.cpp on lines whose row blocks have all of their sequence's units.
#define CX_UNIFORM(x) (x)
#include "cx_share.hpp"

namespace cx {
template <int TOK, int NT>
using TreeLine = AttendLine<TOK, NT, true>;
}
#define AttendLine TreeLine
#define share_split(line, workers) share_split(line, workers, 2)
#define main share_check_main
#include "share_check.cpp"
#undef main

// A row block's units are its sequence's, whatever its rows.
template <int NT>
static bool whole(const Batch& x) {
  using Line = TreeLine<32, NT>;
  for (size_t b = 0; b < x.len.size(); ++b) {
    const AttendSeq s = Line::seq(x.A, x.start[b], x.start[b + 1], x.len[b]);
    if (s.q <= 0 || s.n <= 0) continue;
    const uint64_t one = line_units(Line::length(x.A, s));
    const uint64_t blocks = (uint64_t)Line::row_blocks(x.A, s) * x.A.heads;
    CHECK(one % blocks == 0 && one / blocks >= (uint64_t)s.n, "%lu units of %lu row blocks",
          (unsigned long)one, (unsigned long)blocks);
  }
  return true;
}

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? atoi(argv[1]) : 300;
  rng.seed(argc > 2 ? atoi(argv[2]) : 1);
  long n = 0;
  for (int i = 0; i < rounds; ++i)
    for (int kind = 0; kind < 7; ++kind) {
      const Batch x = make(kind);
      bool ok;
      switch ((i + kind) % 4) {
        case 0: ok = check<32, 2>(x) && whole<2>(x); break;
        case 1: ok = check<32, 4>(x) && whole<4>(x); break;
        case 2: ok = check<32, 8>(x) && whole<8>(x); break;
        default: ok = check<32, 16>(x) && whole<16>(x);
      }
      if (!ok) return 1;
      ++n;
    }
  if (!fixed<32, 2>() || !fixed<32, 16>()) return 1;
  printf("ok %ld\n", n);
}
