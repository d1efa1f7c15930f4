// Checks AddUpTo (kernels/kv_element.h), the sums by which the paged operators'
// kernels share out work that device arrays name, on the CPU: with starts that
// give thousands of sequences the same millions of tokens, each place of the grid
// still belongs to one sequence at most. And WorkerAt (kernels/attend.h), the
// order in which a grid's workgroups take attention's parts.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "attend.h"
#include "kv_element.h"

using kvx::AddUpTo;

static_assert(AddUpTo(0, 0, 0) == 0 && AddUpTo(3, 4, 8) == 7 && AddUpTo(4, 4, 8) == 8, "");
static_assert(AddUpTo(8, 8, 8) == 8 && AddUpTo(INT_MAX, INT_MAX, INT_MAX) == INT_MAX, "");
static_assert(AddUpTo(INT_MAX, 1, INT_MAX) == INT_MAX, "");

// Every worker has one place, an XCD's (every eighth place) are neighbours, and no
// XCD has more than its share: a grid that was sized for longer sequences than
// the call has leaves no XCD idle.
bool Places(int grid, int workers) {
  std::vector<int> place(workers, -1);
  int of[8] = {0}, low[8], high[8];
  for (int x = 0; x < 8; ++x) {
    low[x] = INT_MAX;
    high[x] = -1;
  }
  for (int p = 0; p < grid; ++p) {
    const int w = kvx::WorkerAt(p, workers);
    if (w < 0) continue;
    if (w >= workers || place[w] >= 0) return false;
    place[w] = p;
    ++of[p % 8];
    low[p % 8] = w < low[p % 8] ? w : low[p % 8];
    high[p % 8] = w > high[p % 8] ? w : high[p % 8];
  }
  for (int w = 0; w < workers; ++w) {
    if (place[w] < 0) return false;
  }
  for (int x = 0; x < 8; ++x) {
    if (of[x] > (workers + 7) / 8) return false;
    if (of[x] > 0 && high[x] - low[x] + 1 != of[x]) return false;
  }
  return true;
}

int main() {
  for (int grid : {256, 512}) {
    for (int workers = 0; workers <= grid; ++workers) {
      if (!Places(grid, workers)) {
        std::printf("FAIL: %d workers in a grid of %d\n", workers, grid);
        return 1;
      }
    }
  }
  // Sequence 2 k has all of `each` tokens, sequence 2 k + 1 none; a block a token.
  for (int each : {1, 4096, (1 << 20) + 1, (1 << 21) + 2048, 1 << 29}) {
    const int grid = each;
    int64_t owners = 0;  // of the grid's places
    int before = 0, last = 0;
    for (int s = 0; s < 4096; ++s) {
      const int n = s % 2 == 0 ? each : 0;
      if (before < 0 || before > grid || before < last) {
        std::printf("FAIL: %d blocks each, sequence %d starts at %d\n", each, s, before);
        return 1;
      }
      // The places [before, before + n) of the grid.
      owners += AddUpTo(before, n, grid) - before;
      last = before;
      before = AddUpTo(before, n, grid);
    }
    if (owners != grid) {
      std::printf("FAIL: %lld owners of %d places\n", static_cast<long long>(owners), grid);
      return 1;
    }
  }
  // Valid work is summed as it is, in any grouping.
  const std::vector<int> work = {5, 0, 17, 1, 1, 90, 3};
  const int most = 120;
  for (size_t cut = 0; cut <= work.size(); ++cut) {
    int a = 0, b = 0, plain = 0;
    for (size_t i = 0; i < work.size(); ++i) {
      int& side = i < cut ? a : b;
      side = AddUpTo(side, work[i], most);
      plain += work[i];
    }
    if (AddUpTo(a, b, most) != plain || AddUpTo(a, b, 50) != 50) {
      std::printf("FAIL: sums of %zu and %zu terms\n", cut, work.size() - cut);
      return 1;
    }
  }
  std::printf("paged sums: all passed\n");
  return 0;
}
