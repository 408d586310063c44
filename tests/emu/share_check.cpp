// The split of attention batches over workers (cx_share.hpp), as attend_split
// walks it, on random batches: every unit that a row block's rows may attend to is
// in exactly one piece, in order; the parts of a cut row block are those of
// consecutive workers, and one join entry in range names them.  The lengths and first
// rows in "device memory" change as soon as the workgroup has read them.
#define CX_UNIFORM(x) (x)
#include "cx_share.hpp"

#include <map>
#include <random>
#include <tuple>

using namespace cx;

static std::mt19937_64 rng;
static int64_t pick(int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); }
static int64_t spread(int64_t lo, int64_t hi) {      // over the logarithm
  return std::min<int64_t>(hi, (int64_t)(lo * std::exp((rng() % 100000) / 1e5 * std::log((hi + 1.0) / lo))));
}

struct Batch {
  ShareBatch A;
  std::vector<int> start, len;
  unsigned workers;
  const char* kind;
};

static void print(const Batch& x) {
  printf("%s: G %d heads %d window %d held %d workers %u B %zu", x.kind, x.A.G, x.A.heads, x.A.window,
         x.A.held, x.workers, x.len.size());
  for (size_t b = 0; b < x.len.size() && b < 6; ++b) printf(" (%d of %d)", x.start[b + 1] - x.start[b], x.len[b]);
  printf("\n");
}
#define CHECK(c, ...)                                       \
  if (!(c)) {                                               \
    printf("line %d: %s: ", __LINE__, #c), printf(__VA_ARGS__), printf("\n"), print(x); \
    return false;                                           \
  }

template <int TOK, int NT>
static bool check(const Batch& x) {
  using Line = AttendLine<TOK, NT>;
  const int B = (int)x.len.size();
  std::vector<int> kv_len = x.len, q_start = x.start;
  bool starts = rng() % 2;
  for (int b = 0; b <= B; ++b) starts |= x.start[b] != b;
  std::vector<uint64_t> store(AttendSeqs<uint64_t*, int*>::bytes(B, starts) / 8 + 1);
  uint64_t* const pref = store.data();
  int* const len = (int*)(pref + B + 1);
  const AttendSeqs<uint64_t*, int*> at = {pref, len, len + B, starts};
  for (int tid = 0; tid < 256; ++tid)
    at.read(kv_len.data(), starts ? q_start.data() : nullptr, B, x.start.back(), tid, 256);
  for (int& n : kv_len) n = (int)rng();
  for (int& n : q_start) n = (int)rng();
  auto seq = [&](int b) { return Line::seq(x.A, at.first(b), at.end(b), at.len[b]); };
  std::vector<AttendSeq> seqs(B);
  pref[0] = 0;
  for (int b = 0; b < B; ++b) {
    seqs[b] = Line::seq(x.A, x.start[b], x.start[b + 1], x.len[b]);
    pref[b + 1] = pref[b] + Line::length(x.A, seq(b));
  }
  const uint64_t line = pref[B];
  const ShareSplit split = share_split(line, x.workers);
  const size_t entries = split.by_block ? line_blocks(line) : x.workers;
  CHECK(entries <= x.workers, "%zu entries", entries);
  std::vector<AttendJoin> join(entries);
  std::vector<char> written(entries, 0);
  struct Part { int unit, cnt, slot; unsigned worker; };
  std::map<std::tuple<int, int, int>, std::vector<Part>> parts;
  uint64_t next = 0;
  for (unsigned w = 0; w < x.workers && w < split.shares; ++w) {
    uint64_t u = share_begin(split, w);
    const uint64_t end = u + split.per + (w < split.more);
    CHECK(u == next && end > u, "worker %u", w);
    next = end;
    int b = 0;
    for (int hi = B - 1; b < hi;) {
      const int mid = (b + hi + 1) >> 1;
      if (line_units(pref[mid]) <= u) b = mid;
      else hi = mid - 1;
    }
    while (u < end) {
      while (line_units(pref[b + 1]) <= u) ++b;
      CHECK(b < B, "sequence %d", b);
      const uint64_t u0 = u;
      bool fine = true;
      const AttendPiece p = Line::piece(x.A, seq(b), b, pref[b], split, w, end, u,
                                        [&](unsigned entry, const AttendJoin& j) {
        fine = entry < entries && !written[entry];
        if (!fine) return;
        written[entry] = 1;
        join[entry] = j;
      });
      CHECK(fine, "an entry out of range, or twice");
      CHECK(u > u0 && u <= end, "no progress at %lu", (unsigned long)u0);
      if (p.cnt == 0) { CHECK(u == end, "an empty piece inside a share"); break; }
      CHECK(p.cnt > 0 && p.h >= 0 && p.h < x.A.heads && p.r0 >= 0 && p.r0 % Line::ROWS == 0 &&
            p.R >= 1 && p.R <= Line::ROWS && p.r0 + p.R <= seqs[b].q * x.A.G,
            "cnt %d head %d rows %d + %d", p.cnt, p.h, p.r0, p.R);
      CHECK(p.tok0 == x.start[b] && p.lowest == seqs[b].len - seqs[b].q && p.lim == seqs[b].lim, "piece");
      parts[{b, p.h, p.r0}].push_back({p.unit, p.cnt, p.slot, w});
    }
  }
  CHECK(next == line_units(line), "%lu of %lu units", (unsigned long)next, (unsigned long)line_units(line));
  std::map<std::tuple<int, int, int>, const AttendJoin*> joined;
  for (size_t e = 0; e < entries; ++e) {
    if (!written[e]) { CHECK(!split.by_block, "row block %zu has no entry", e); continue; }
    if (join[e].last < 0) continue;
    const AttendJoin& J = join[e];
    CHECK(J.first >= 0 && J.last >= J.first && J.last < (int)x.workers, "entry %zu", e);
    int b = 0;
    while (!(x.start[b] == J.tok0 && x.start[b + 1] > J.tok0)) ++b;
    CHECK(joined.emplace(std::tuple{b, J.head, J.row0}, &J).second, "two entries");
  }
  for (int b = 0; b < B; ++b) {
    const AttendSeq& s = seqs[b];
    const int blocks = s.q > 0 ? Line::row_blocks(x.A, s) : 0;
    for (int h = 0; h < x.A.heads; ++h)
      for (int rb = 0; rb < blocks; ++rb) {
        const auto it = parts.find({b, h, rb * Line::ROWS});
        const int64_t lowest = (int64_t)s.len - s.q, rows = (int64_t)s.q * x.A.G;
        const int64_t low = lowest + (int64_t)rb * Line::ROWS / x.A.G,
                      high = lowest + (std::min<int64_t>((rb + 1LL) * Line::ROWS, rows) - 1) / x.A.G;
        const int64_t from = x.A.window ? std::max<int64_t>(low - x.A.window + 1, 0) : 0,
                      to = std::min<int64_t>(high + 1, s.lim);
        if (it == parts.end()) {
          CHECK(to <= from || s.n <= 0, "row block %d of sequence %d is nowhere", rb, b);
          CHECK(s.n <= 0, "row block %d of sequence %d is not written", rb, b);
          continue;
        }
        const auto& v = it->second;
        if (to > from) {
          CHECK(v.front().unit <= from / TOK, "starts at %d, not %ld", v.front().unit, (long)(from / TOK));
          CHECK((int64_t)v.back().unit + v.back().cnt >= (to + TOK - 1) / TOK, "ends early");
        }
        for (size_t k = 1; k < v.size(); ++k) {
          CHECK(v[k].unit == v[k - 1].unit + v[k - 1].cnt && v[k].worker == v[k - 1].worker + 1, "order");
        }
        const auto j = joined.find(it->first);
        if (v.size() == 1) {
          CHECK(v[0].slot == -1 && j == joined.end(), "slot %d of a whole row block", v[0].slot);
          continue;
        }
        CHECK(j != joined.end(), "cut, not joined");
        const AttendJoin& J = *j->second;
        CHECK(J.first == (int)v.front().worker && J.last == (int)v.back().worker, "workers %d .. %d",
              J.first, J.last);
        CHECK(J.rows == std::min<int64_t>(Line::ROWS, rows - rb * Line::ROWS), "rows %d", J.rows);
        for (size_t k = 0; k < v.size(); ++k)
          CHECK(v[k].slot == 2 * (J.first + (int)k) + (k == 0), "slot %d of part %zu", v[k].slot, k);
      }
  }
  CHECK(joined.size() <= parts.size(), "entries of nothing");
  return true;
}

static Batch make(int kind) {
  static const char* names[] = {"decode", "many", "verify", "prompts", "mixed", "edges", "one long"};
  Batch x;
  x.kind = names[kind];
  x.A.G = (int)pick(1, kind == 3 ? 8 : 12);
  x.A.heads = (int)pick(1, 8);
  x.A.window = pick(0, 2) ? 0 : (int)spread(1, 3000);
  x.workers = (unsigned)(pick(0, 3) ? 1024 << pick(0, 2) : 4 * pick(1, 200));
  int B = kind == 1 ? (int)pick(513, 4096) : (int)spread(1, 200);
  int64_t cap = kind == 1 ? 80 : kind == 6 ? 200000 : 5000;
  if (kind == 3 || kind == 6) B = (int)pick(1, 4);
  if (kind == 1) x.A.heads = (int)pick(1, 2);
  x.start.push_back(0);
  int64_t most = 1;
  for (int b = 0; b < B; ++b) {
    int64_t len = pick(0, 9) ? spread(1, cap) : 0, q = 1;
    if (kind == 2) q = pick(1, 9);
    if (kind == 3) q = std::max<int64_t>(1, spread(1, 2000));
    if (kind == 4 || kind == 5) q = pick(0, 3) ? pick(0, 9) : spread(1, 600);
    if (kind == 5) len = pick(0, 2) ? pick(-5, 700) : (int64_t)INT32_MAX - pick(0, 100);
    if (kind != 5 && pick(0, 19)) q = std::min(q, std::max<int64_t>(len, 1));
    x.start.push_back((int)(x.start.back() + q));
    x.len.push_back((int)len);
    most = std::max(most, len);
  }
  x.A.held = (int)(pick(0, 3) || kind == 5 ? std::min<int64_t>(most, 16 * pick(0, 300)) : (most + 15) / 16 * 16);
  if (!pick(0, 30)) x.A.held = 0;
  return x;
}

template <int TOK, int NT>
static bool fixed() {
  // more row blocks in a sequence than workers, its rows' positions from 0 on
  Batch x{{1, 64, 0, 2048}, {0, 1030}, {1030}, 4096, "hint of one"};
  // a prompt at the last positions
  Batch y{{2, 1, 0, 4096}, {0, 70}, {INT32_MAX}, 1024, "last positions"};
  return check<TOK, NT>(x) && check<TOK, NT>(y);
}

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? atoi(argv[1]) : 300;
  rng.seed(argc > 2 ? atoi(argv[2]) : 1);
  long n = 0;
  for (int i = 0; i < rounds; ++i)
    for (int kind = 0; kind < 7; ++kind) {
      const Batch x = make(kind);
      bool ok;
      switch ((i + kind) % 6) {
        case 0: ok = check<32, 1>(x); break;
        case 1: ok = check<32, 2>(x); break;
        case 2: ok = check<32, 3>(x); break;
        case 3: ok = check<32, 4>(x); break;
        case 4: ok = check<64, 1>(x); break;
        default: ok = check<64, 2>(x);
      }
      if (!ok) return 1;
      ++n;
    }
  if (!fixed<32, 1>() || !fixed<64, 1>()) return 1;
  printf("ok %ld\n", n);
}
