// The columns of the few-rows product's groups (csrc/mx_columns.hpp), built for the host:
// test_mx_columns.py goes through every group of a launch.
#include "../../npu-dialect_amd/csrc/mx_columns.hpp"

using namespace npu;

extern "C" {

// Of N columns in groups of 16 nt: how often each is stored (stored[N]), and by how far the vectors of
// the workspace lie off 16 bytes or past their row (off).  Returns the rows of w read outside [0, N), -1 if
// a column is computed from another row.
int mx_columns(int N, int nt, int *stored, int *off) {
  const long long width = (N + 3LL) & ~3LL;
  int outside = 0;
  *off = 0;
  for (int i = 0; i < (N + 16 * nt - 1) / (16 * nt); ++i) {
    const FewColumns c(i, nt, N);
    for (int t = 0; t < nt; ++t) {
      for (int r = 0; r < 16; ++r) {
        const long long row = c.n0 + c.row(t, r);
        if (row < 0 || row >= N) ++outside;
      }
      for (int g = 0; g < 4; ++g) {
        const long long n = c.first(t, g);
        if (n >= N) continue;
        if (n % 4 != 0 || n < 0 || n + 4 > width) ++*off;
        for (int e = 0; e < 4 && n + e < N; ++e) {
          ++stored[n + e];
          // (the instruction leaves row 4 g + e of the tile there)
          if (c.n0 + c.row(t, 4 * g + e) != n + e) return -1;
        }
      }
    }
  }
  return outside;
}

}  // extern "C"
