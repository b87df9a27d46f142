// Launches in two dimensions (csrc/nls_tile.h) on the host: for every number of workgroups up to 2^31 rows can ask for, the grid holds them all, its rows are
// whole, and no dimension has more threads or workgroups than a launch counts.
#include <cstdio>

#include "nls_tile.h"

template <int THREADS>
int check(long groups) {
  const dim3 g = lb::grid_of<THREADS>(groups);
  const bool fine = (long)g.x * THREADS < 1l << 32 && g.y <= 65535 && g.z == 1 && (long)g.x * g.y >= groups && (long)g.x * (g.y - 1) < groups &&
                    (g.y == 1 || g.x == lb::GRID_X);
  if (!fine) std::printf("%ld workgroups of %d threads: %u x %u\n", groups, THREADS, g.x, g.y);
  return fine ? 0 : 1;
}

int main() {
  int wrong = 0;
  for (int e = 0; e <= 31; ++e)
    for (long d = -33; d <= 33; ++d) {
      const long groups = (1l << e) + d;
      if (groups < 1 || groups > 1l << 31) continue;
      wrong += check<256>(groups) + check<512>(groups) + check<1024>(groups);
    }
  wrong += check<1024>((1l << 27) / 32) + check<1024>(((1l << 31) - 1 + 31) / 32);  // 32 rows of a transposed matrix a workgroup
  std::printf("wrong: %d\n", wrong);
  return wrong != 0;
}
